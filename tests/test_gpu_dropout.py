"""counter_dropout: the mask bit for bit, its rate, values that are not finite, strides, graphs."""
import pytest
import torch

import pack3d_amd as p3d
from tests._block_reference import keep_mask

pytestmark = pytest.mark.gpu


def _expected(x, p, seed, offset):
    threshold = min(65535, int(p * 65536 + 0.5))
    keep = keep_mask(x.numel(), threshold, seed, offset).view(x.shape)
    # one product in fp32 with the fp32 reciprocal of the share that stays, rounded to x's type
    inv = torch.tensor(65536.0, dtype=torch.float32) / torch.tensor(65536.0 - threshold, dtype=torch.float32)
    return torch.where(keep, (x.float() * inv), 0.0).to(x.dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (2047,), (2048,), (2049,), (3, 5, 11), (100003,), (1, 4096, 64)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_values_and_gradient(gpu, dtype, shape, p):
    gen = torch.Generator().manual_seed(len(shape))
    x, dy = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
    seed, offset = 0x7EDCBA9876543210, 0x123456789
    xd = x.to(gpu).requires_grad_()
    y = p3d.counter_dropout(xd, p, (seed, offset))
    assert torch.equal(y.cpu(), _expected(x, p, seed, offset))
    (dx,) = torch.autograd.grad(y, xd, dy.to(gpu))
    assert torch.equal(dx.cpu(), _expected(dy, p, seed, offset))
    state = torch.tensor([seed, offset], device=gpu)
    with torch.no_grad():
        assert torch.equal(p3d.counter_dropout(xd, p, state), y)
        assert not torch.equal(p3d.counter_dropout(xd, p, (seed, offset + 1)), y) or x.numel() < 20


def test_the_generator_gives_its_published_values():
    """The first block of Philox4x32-10 for a zero counter and key, as the generator's paper publishes it:
    6627e8d5 e169c58d bc57ac4c 9b00dbd8."""
    halves = []
    for word in (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8):
        halves += [word & 0xFFFF, word >> 16]
    for threshold in range(0, 65536, 257):
        assert keep_mask(8, threshold, 0, 0).tolist() == [h >= threshold for h in halves]


@pytest.mark.parametrize("p", [2.0 ** -16, 0.01, 0.1, 0.9, 1 - 2.0 ** -16])
def test_rate(gpu, p):
    """The share dropped of 4M elements within six standard deviations of the rate."""
    n = 1 << 22
    y = p3d.counter_dropout(torch.ones(n, device=gpu), p, 77)
    share = (y == 0).double().mean().item()
    assert abs(share - p) <= 6 * (p * (1 - p) / n) ** 0.5
    assert abs(y.double().mean().item() - 1) <= 6 * (p / (1 - p) / n) ** 0.5 + 1e-6


def test_what_is_dropped_may_be_anything(gpu):
    keep = keep_mask(4096, 32768, 3, 0).to(gpu)
    x = torch.where(keep, 1.0, float("nan"))
    assert torch.equal(p3d.counter_dropout(x, 0.5, 3), torch.where(keep, 2.0, 0.0))
    x = torch.where(keep, float("inf"), 1.0)
    assert torch.equal(p3d.counter_dropout(x, 0.5, 3) == float("inf"), keep)


def test_strides_do_not_matter(gpu):
    x = torch.randn(40, 3, 21, device=gpu)
    t = x.permute(2, 0, 1)
    assert torch.equal(p3d.counter_dropout(t, 0.3, 5), p3d.counter_dropout(t.contiguous(), 0.3, 5))
    part = x[:, 1]
    assert torch.equal(p3d.counter_dropout(part, 0.3, 5), p3d.counter_dropout(part.contiguous(), 0.3, 5))
    assert p3d.counter_dropout(x[:0], 0.3, 5).shape == (0, 3, 21)
    assert p3d.counter_dropout(x, 0.0, None) is x
    odd = torch.randn(1001, device=gpu)[1:]
    assert torch.equal(p3d.counter_dropout(odd, 0.3, 5), p3d.counter_dropout(odd.clone(), 0.3, 5))


def test_same_mask_as_the_block(gpu):
    """block_residual applies the same mask inside, at widths that divide into groups of eight and that do not."""
    for dim in (48, 77):
        x, y = (torch.randn(2, 19, dim, device=gpu) for _ in range(2))
        out = p3d.block_residual(torch.zeros_like(x), y, p=0.4, seed=(12, 3))
        assert torch.equal(out, p3d.counter_dropout(y, 0.4, (12, 3)))


def test_in_a_graph_with_a_seed_per_replay(gpu):
    x = torch.randn(5000, device=gpu)
    seed = torch.tensor([1, 0], device=gpu)
    p3d.counter_dropout(x, 0.3, seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = p3d.counter_dropout(x, 0.3, seed)
        seed[1].add_(1)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, p3d.counter_dropout(x, 0.3, (1, i)))
