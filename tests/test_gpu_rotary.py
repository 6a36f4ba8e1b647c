"""apply_rotary against its definition in 64 bits.

The kernel forms the angle in turns in 64 bits and rounds its distance from a whole
turn to fp32 (at most 2^-26 turns, 2 pi 2^-26 < 2^-23 radians), then sin and cos (2
units of 2^-24 each at most 1), times magnitude: each of them is off by at most 2^-23 +
3 * 2^-24 < 6 U relative to magnitude; two products and a sum add 3 U."""
import math

import pytest
import torch

import pack3d_amd as p3d
from tests._block_reference import U, assert_within, half_step, rotary_reference, smallest

pytestmark = pytest.mark.gpu


def _check(got, x, ref, magnitude, pairs, layout, name):
    p = sum(pairs)
    size = x.double().abs()
    if layout == "half":
        both = size[..., :p] + size[..., p:2 * p]
        both = torch.cat((both, both), -1)
    else:
        both = (size[..., 0:2 * p:2] + size[..., 1:2 * p:2]).repeat_interleave(2, -1)
    bound = torch.cat((both * magnitude * 9 * U, torch.zeros_like(size[..., 2 * p:])), -1)
    bound = bound + half_step(got.dtype) * (ref.abs() + bound) + smallest(got.dtype)
    assert_within(got, ref, bound, name)
    assert torch.equal(got[..., 2 * p:].cpu(), x[..., 2 * p:])


def _run(gpu, b, heads, n, d, pairs, layout, dtype, positions, magnitude=1.0, scaling="none", views=False):
    gen = torch.Generator().manual_seed(n + d)
    freqs, _ = p3d.rotary_frequencies(pairs, scaling=scaling, factor=4.0, trained=1024.0)
    xs = [torch.randn(b, n, h, d, generator=gen).to(dtype).transpose(1, 2) for h in heads]
    ups = [torch.randn(b, h, n, d, generator=gen).to(dtype) for h in heads]
    dev = [t.to(gpu) if views else t.to(gpu).contiguous() for t in xs]
    dev = [t.requires_grad_() for t in dev]
    pos3 = positions if len(pairs) > 1 else positions.unsqueeze(-1)
    pos3 = pos3 if pos3.ndim == 3 else pos3.unsqueeze(0)
    outs = p3d.apply_rotary(dev, positions.to(gpu), freqs.to(gpu), pairs=pairs, layout=layout, magnitude=magnitude)
    grads = torch.autograd.grad(outs, dev, [u.to(gpu) for u in ups])
    for x, out, up, g in zip(xs, outs, ups, grads):
        _check(out, x, rotary_reference(x, pos3, freqs, pairs, layout, magnitude), magnitude, pairs, layout, "out")
        _check(g, up, rotary_reference(up, pos3, freqs, pairs, layout, magnitude, inverse=True), magnitude, pairs,
               layout, "grad")
    with torch.no_grad():
        for a, b_ in zip(p3d.apply_rotary(dev, positions.to(gpu), freqs.to(gpu), pairs=pairs, layout=layout,
                                          magnitude=magnitude), outs):
            assert torch.equal(a, b_)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("d,pairs", [(16, 8), (16, 3), (48, 24), (64, 32), (64, 16), (80, 37), (128, 64), (128, 1),
                                     (2, 1), (7, 3), (15, 7), (16, 7), (17, 1), (24, 5), (20, 8), (40, 4),
                                     (33, 13), (256, 128), (1024, 512)])
def test_heads_and_layouts(gpu, dtype, layout, d, pairs):
    _run(gpu, 2, (4, 2), 29, d, (pairs,), layout, dtype, torch.arange(29) * 3)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_axes(gpu, layout):
    side = torch.stack(torch.meshgrid(*(torch.arange(k) for k in (3, 5, 4)), indexing="ij"), -1).reshape(-1, 3)
    _run(gpu, 2, (4, 2, 2), 60, 48, (8, 8, 8), layout, torch.bfloat16, side, scaling="linear", views=True)
    _run(gpu, 1, (4,), 60, 48, (9, 0, 7), layout, torch.float32, side.to(torch.int32), scaling="parts", magnitude=1.2)
    _run(gpu, 1, (4,), 60, 32, (8, 8), layout, torch.float32, side[:, 1:], scaling="ntk")
    _run(gpu, 2, (1,), 60, 32, (5, 5, 5), layout, torch.float16, torch.stack((side, side.flip(0))))


@pytest.mark.parametrize("first", [0, 1_000_000, 2 ** 31 - 100, -5, 2 ** 40])
def test_far_positions(gpu, first):
    """Positions far out keep their angles: in 64 bits the angle of 2^40 is off by 2^40 2^-52 radians times a few,
    below 2^-9; closer ones by less than the fp32 rounding that the bound counts."""
    n = 33
    positions = first + torch.arange(n)
    if abs(first) <= 2 ** 31:
        _run(gpu, 1, (2,), n, 64, (32,), "half", torch.float32, positions)
    else:
        freqs, _ = p3d.rotary_frequencies(32)
        x = torch.randn(1, 2, n, 64, generator=torch.Generator().manual_seed(1))
        out = p3d.apply_rotary(x.to(gpu), positions.to(gpu), freqs.to(gpu))
        ref = rotary_reference(x, positions.view(1, n, 1), freqs, (32,), "interleaved", 1.0)
        # the product of position and frequency is off by half a step of 2^40 in each of the two forms, and 1 / 2 pi adds one
        assert (out.double().cpu() - ref).abs().max() <= 4 * 2 ** 40 * 2 ** -53 * x.abs().max() * 1.5


@pytest.mark.parametrize("b,n,heads", [(8, 1, (8, 2)), (1, 1, (1,)), (3, 2, (64, 8)), (1, 5000, (4, 4, 4)), (1, 1, (500,)),
                                       (4, 257, (3,))])
def test_tokens_and_batches(gpu, b, n, heads):
    gen = torch.Generator().manual_seed(2)
    positions = torch.randint(0, 100000, (b, n), generator=gen)
    _run(gpu, b, heads, n, 64, (32,), "half", torch.bfloat16, positions, views=True)
    _run(gpu, b, heads, n, 40, (17,), "interleaved", torch.float32, positions.to(torch.int32))


def test_strides(gpu):
    """Views at odd offsets, expanded heads, transposed positions and expanded gradients."""
    n, d = 21, 32
    wide = torch.randn(2, n, 4 * d + 3, device=gpu)
    x = wide[..., 3:].view(2, n, 4, d).transpose(1, 2) if wide[..., 3:].is_contiguous() else \
        wide[..., 3:].unflatten(-1, (4, d)).transpose(1, 2)
    positions = torch.randint(0, 999, (n, 2), device=gpu).t()
    freqs = p3d.rotary_frequencies(13)[0].to(gpu)
    shared = x[:, :1].expand(2, 4, n, d)
    swapped = x.transpose(-1, -2).contiguous().transpose(-1, -2)
    for t in (x, shared, swapped):
        a = p3d.apply_rotary(t, positions, freqs)
        assert torch.equal(a, p3d.apply_rotary(t.contiguous(), positions.contiguous(), freqs))
    leaf = x.detach().requires_grad_()
    out = p3d.apply_rotary(leaf, positions, freqs)
    (g,) = torch.autograd.grad(out.sum(), leaf)
    leaf2 = x.detach().requires_grad_()
    (g2,) = torch.autograd.grad(p3d.apply_rotary(leaf2, positions, freqs), leaf2, torch.ones_like(out))
    assert torch.equal(g, g2)
    assert p3d.apply_rotary(x[:0], positions[:1], freqs).shape == (0, 4, n, d)


def test_rows_beyond_four_gigabytes(gpu):
    """Tokens 8 MiB apart read as a contiguous copy of them does."""
    n, stride = 1100, 1 << 22
    x = torch.empty(n * stride, dtype=torch.bfloat16, device=gpu).as_strided((1, 2, n, 64), (0, 64, stride, 1))
    x.copy_(torch.randn(1, 2, n, 64, device=gpu))
    positions, freqs = torch.arange(n, device=gpu), p3d.rotary_frequencies(20)[0].to(gpu)
    assert torch.equal(p3d.apply_rotary(x, positions, freqs, layout="half"),
                       p3d.apply_rotary(x.contiguous(), positions, freqs, layout="half"))


def test_some_gradients_only(gpu):
    q, k = (torch.randn(1, 2, 9, 16, device=gpu) for _ in range(2))
    k.requires_grad_()
    freqs = p3d.rotary_frequencies(8)[0].to(gpu)
    positions = torch.arange(9, device=gpu)
    a, b = p3d.apply_rotary((q, k), positions, freqs, layout="half")
    up = torch.randn_like(b)
    (g,) = torch.autograd.grad(b, k, up)
    (alone,) = torch.autograd.grad(p3d.apply_rotary(k, positions, freqs, layout="half"), k, up)
    assert torch.equal(g, alone)


def test_gradient_agrees_with_differences(gpu):
    """Turning is linear: <dout, R(x + h d) - R(x - h d)> / 2h = <R^T dout, d> in 64 bits up to rounding, which the
    gradient's fp32 bound covers (9 U of the terms' magnitudes)."""
    gen = torch.Generator().manual_seed(3)
    x, up, step = (torch.randn(1, 2, 11, 24, generator=gen) for _ in range(3))
    freqs = p3d.rotary_frequencies((4, 4, 2))[0]
    positions = torch.randint(0, 50, (11, 3), generator=gen)
    leaf = x.to(gpu).requires_grad_()
    out = p3d.apply_rotary(leaf, positions.to(gpu), freqs.to(gpu), pairs=(4, 4, 2))
    (g,) = torch.autograd.grad(out, leaf, up.to(gpu))

    def turned(t):
        return rotary_reference(t.double(), positions.view(1, 11, 3), freqs, (4, 4, 2), "interleaved", 1.0)
    difference = (up.double() * (turned(x.double() + 0.5 * step.double()) - turned(x.double() - 0.5 * step.double()))).sum()
    terms = g.double().cpu() * step.double()
    assert abs(terms.sum() - difference) <= 9 * U * 2 * (up.abs().double() * step.abs().double()).sum() * 4


def test_in_a_graph(gpu):
    x = torch.randn(2, 3, 1, 64, device=gpu)
    positions = torch.tensor([[3], [900]], device=gpu)
    freqs = p3d.rotary_frequencies(32)[0].to(gpu)
    p3d.apply_rotary(x, positions, freqs, layout="half")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = p3d.apply_rotary(x, positions, freqs, layout="half")
        positions.add_(1)
    for i in range(3):
        now = positions.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, p3d.apply_rotary(x, now, freqs, layout="half"))


def test_frequencies():
    """Interpolated by the factor, the base raised so that the slowest pair alone is, and by parts between the two."""
    plain, one = p3d.rotary_frequencies(16)
    assert one == 1.0 and torch.allclose(plain, 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16), rtol=1e-14)
    assert torch.equal(p3d.rotary_frequencies(16, scaling="linear", factor=4.0)[0], plain / 4)
    ntk = p3d.rotary_frequencies(16, scaling="ntk", factor=4.0)[0]
    assert ntk[0] == 1 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12) and (ntk[1:] < plain[1:]).all()
    parts, m = p3d.rotary_frequencies(64, scaling="parts", factor=4.0, trained=2048)
    plain = p3d.rotary_frequencies(64)[0]
    assert math.isclose(m, 0.1 * math.log(4) + 1)
    turns = 2048 * plain / (2 * math.pi)
    assert torch.equal(parts[turns > 32], plain[turns > 32]) and torch.equal(parts[turns < 1], plain[turns < 1] / 4)
    assert torch.equal(p3d.rotary_frequencies((5, 0, 3))[0], torch.cat((p3d.rotary_frequencies(5)[0],
                                                                       p3d.rotary_frequencies(3)[0])))
