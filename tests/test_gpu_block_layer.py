"""The operators around a block together, as the layer calls them: two layers with rotary positions, a post norm,
scale, dropout and gates, the first handing the second its normalised input, against the oracle's core and plain
operations in 64 bits on the CPU, outputs and every gradient.

Tolerances are of the 2-norm of a tensor's difference over its norm.  fp32: a value goes through about 30 sums of at most
192 terms (each off by at most 200 * 2^-24 of its terms' magnitudes, in practice its square root), norms and products:
30 * sqrt(200) * 2^-24 = 2.6e-5, doubled twice for cancellation in the norms' gradients: 1e-4.  bf16: 30 roundings of
2^-9 (root mean square of at most 2^-8), adding as squares: sqrt(30) * 2^-9 = 0.011, times three: 0.035, the bar of the
layer's other tests."""
import math

import pytest
import torch

import oracle.pack3d_oracle as ref
import pack3d_amd as p3d
from tests._block_reference import keep_mask, rotary_reference
from tests._cases import rel_l2

pytestmark = pytest.mark.gpu

SHAPE, DIM, HEADS, KV, HEAD_DIM = (4, 8, 8), 96, 4, 2, 32


def _layers(encoding, rotary, dropout=0.0, post=("rms", "layer")):
    torch.manual_seed(3)
    layers = [p3d.PACK3DAttention(DIM, heads=HEADS, kv_heads=KV, head_dim=HEAD_DIM, block_volume=64,
                                  position_encoding=encoding, rotary=rotary, post_norm=kind, layer_scale=scale,
                                  dropout=dropout) for kind, scale in zip(post, (0.5, None))]
    for layer in layers:  # parameters that do something
        with torch.no_grad():
            for name, q in layer.named_parameters():
                if "norm" in name:
                    q.add_(0.1 * torch.randn(q.shape))
    return layers


def _plain(p, x, layout, encoding, rotary, gate, keep, normed=None):
    """One block of parameters p in x's type (64 bits) with plain operations and the oracle's core."""

    def norm(x, pre, kind, eps=1e-5):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * p[pre + "weight"]
        return x + p[pre + "bias"] if pre + "bias" in p else x
    b, n, _ = x.shape
    xn = norm(x, "norm.", "layer") if normed is None else normed
    q = (xn @ p["to_q.weight"].t()).view(b, n, HEADS, HEAD_DIM).transpose(1, 2)
    kl, vl, kg, vg = ((t.reshape(b, n, KV, HEAD_DIM)).transpose(1, 2) for t in (xn @ p["to_kv.weight"].t()).chunk(4, -1))
    axes = 3 if encoding == "axial" else 1
    positions = layout.coords[None] if axes == 3 else torch.arange(n).view(1, n, 1)
    pairs = rotary.pairs(HEAD_DIM, axes)
    freqs, m = p3d.rotary_frequencies(pairs, base=rotary.base, scaling=rotary.scaling, factor=rotary.factor,
                                      trained=rotary.trained)
    q, kl, kg = (rotary_reference(t, positions, freqs, pairs, rotary.layout, m) for t in (q, kl, kg))
    g = (xn @ p["gate.weight"].t() + p["gate.bias"]).view(b, n, HEADS, 2).softmax(-1)[..., 1].transpose(1, 2)
    o = ref.pack3d_reference(q, kl, vl, kg, vg, p["pool_weight"], p["slot_bias"], g, p["local_scale"], p["global_scale"],
                             layout.geometry)
    y = o.transpose(1, 2).reshape(b, n, -1) @ p["to_out.weight"].t()
    y = norm(y, "post_norm.", "layer" if "post_norm.bias" in p else "rms")
    if keep is not None:
        y = torch.where(keep[0].view(y.shape), y / keep[1], 0.0)
    y = y * gate if gate is not None else y
    return x + (y * p["layer_scale"] if "layer_scale" in p else y)


def _stack(layers, lay, x, gates, final):
    x1, n1 = layers[0](x, lay, residual_gate=gates[0], next_norm=layers[1].norm)
    return layers[1](x1, lay, residual_gate=gates[1], normed=n1, next_norm=final)


CASES = [("axial", p3d.RotaryEncoding(), "fp32", 0.0), ("axial", p3d.RotaryEncoding("half", 0.75, scaling="linear", factor=2.0), "fp32", 0.2),
         ("packed", p3d.RotaryEncoding("half", scaling="parts", factor=4.0, trained=64.0), "fp32", 0.1),
         ("axial", p3d.RotaryEncoding("interleaved", 0.5, scaling="ntk", factor=2.0), "bf16", 0.1),
         ("packed", p3d.RotaryEncoding("half"), "autocast", 0.1)]


@pytest.mark.parametrize("encoding,rotary,dtype,dropout", CASES)
def test_two_blocks(gpu, monkeypatch, encoding, rotary, dtype, dropout):
    print(f"two blocks {encoding} {rotary.layout} {dtype} dropout {dropout}", flush=True)
    layers = _layers(encoding, rotary, dropout)
    n = math.prod(SHAPE)
    gen = torch.Generator().manual_seed(9)
    kind = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = torch.randn(2, n, DIM, generator=gen).to(kind)
    gates = [(0.5 + 0.3 * torch.randn(2, 1, DIM, generator=gen)).to(kind), torch.rand(2, n, 1, generator=gen).to(kind)]
    ups = [torch.randn(2, n, DIM, generator=gen).to(kind) for _ in range(2)]
    layers = [layer.to(kind).train() for layer in layers]
    lay_ref = ref.build_layout(SHAPE, (4, 4, 4), radius=1, pool_size=1, layout="raster_block")
    seeds = [(11, 1), (12, 2)]
    # 64 bits
    t = int(dropout * 65536 + 0.5)
    keeps = [(keep_mask(x.numel(), t, *s), 1 - t / 65536) if t else None for s in seeds]
    states = [{k: v.detach().double().clone().requires_grad_() for k, v in layer.named_parameters()} for layer in layers]
    xr = x.double().requires_grad_()
    gr = [g.double().requires_grad_() for g in gates]
    x1 = _plain(states[0], xr, lay_ref, encoding, rotary, gr[0], keeps[0])
    h = x1 - x1.mean(-1, keepdim=True)
    n1 = h / (h.square().mean(-1, keepdim=True) + 1e-5).sqrt() * states[1]["norm.weight"] + states[1]["norm.bias"]
    x2 = _plain(states[1], x1, lay_ref, encoding, rotary, gr[1], keeps[1], normed=n1)
    n2 = x2 / (x2.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    leaves_r = [xr, *gr, *(v for s in states for v in s.values())]
    grads_r = torch.autograd.grad((x2, n2), leaves_r, [u.double() for u in ups])
    # the layers
    layers = [layer.to(gpu) for layer in layers]
    lay = p3d.build_layout(SHAPE, (4, 4, 4), radius=1, pool_size=1, layout="raster_block", device=gpu)
    given = iter([torch.tensor(s, device=gpu) for s in seeds])
    monkeypatch.setattr("pack3d_amd.attention.new_seed", lambda device: next(given))
    xd = x.to(gpu).requires_grad_()
    gd = [g.to(gpu).requires_grad_() for g in gates]
    with torch.autocast("cuda", torch.bfloat16, enabled=dtype == "autocast"):
        got = _stack(layers, lay, xd, gd, p3d.Norm("rms", eps=1e-6))
    bar = 1e-4 if dtype == "fp32" else 0.035
    for name, a, b in zip(("x2", "n2"), got, (x2, n2)):
        assert a.dtype == (torch.bfloat16 if dtype == "bf16" or (dtype == "autocast" and name == "n2") else torch.float32)
        assert rel_l2(a, b) <= bar, (name, rel_l2(a, b))
    names = ["x", "gate0", "gate1"] + [f"{i}.{k}" for i, s in enumerate(states) for k in s]
    leaves = [xd, *gd, *(v for layer in layers for v in layer.parameters())]
    grads = torch.autograd.grad(got, leaves, [u.to(gpu).to(a.dtype) for u, a in zip(ups, got)])
    for name, a, b in zip(names, grads, grads_r):
        assert a.shape == b.shape and rel_l2(a, b) <= bar, (name, rel_l2(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_normed_input_and_serving_paths(gpu, dtype):
    """Without gradients: the block given its normalised input against the one that normalises, and the end as one pass
    against plain operations on the plain layer's branch.  The normalised input is rounded to dtype where the layer's
    kernel keeps it in that type too; the products sum in another order: 8 roundings of dtype."""
    lay = p3d.build_layout(SHAPE, (4, 4, 4), radius=1, pool_size=1, layout="raster_block", device=gpu)
    plain = p3d.PACK3DAttention(DIM, heads=HEADS, kv_heads=KV, head_dim=HEAD_DIM, block_volume=64).to(gpu, dtype)
    x = torch.randn(1, math.prod(SHAPE), DIM, device=gpu).to(dtype)
    bar = 8 * torch.finfo(dtype).eps
    with torch.no_grad():
        y = plain(x, lay)
        n = p3d.block_norm(x, p3d.Norm.of(plain.norm))
        assert rel_l2(plain(x, lay, normed=n), y) <= bar
        out, after = plain(x, lay, next_norm=torch.nn.RMSNorm(DIM, eps=1e-5, device=gpu))
        assert rel_l2(out, y) <= bar
        wide = y.double()
        assert rel_l2(after, wide / (wide.square().mean(-1, keepdim=True) + 1e-5).sqrt()) <= bar
        gate = torch.full((1, 1, DIM), 0.25, device=gpu, dtype=dtype)
        gated = plain(x, lay, residual_gate=gate)
        assert rel_l2(gated, x.double() + 0.25 * (wide - x.double())) <= bar


def test_dropout_in_training_only(gpu):
    lay = p3d.build_layout(SHAPE, (4, 4, 4), radius=1, pool_size=1, layout="raster_block", device=gpu)
    layer = p3d.PACK3DAttention(DIM, heads=HEADS, kv_heads=KV, head_dim=HEAD_DIM, block_volume=64, dropout=0.5).to(gpu)
    x = torch.randn(1, math.prod(SHAPE), DIM, device=gpu)
    with torch.no_grad():
        layer.eval()
        y = layer(x, lay)
        assert torch.equal(layer(x, lay), y)
        layer.train()
        torch.manual_seed(1)
        a, b = layer(x, lay), layer(x, lay)
        torch.manual_seed(1)
        assert torch.equal(layer(x, lay), a) and not torch.equal(a, b)
        dropped = (a == x).double().mean().item()
        assert abs(dropped - 0.5) <= 6 * 0.5 / x.numel() ** 0.5 + 0.01


def test_serving_block_in_a_graph(gpu):
    """A gated block with rotary positions and the next norm, captured and replayed on new inputs."""
    lay = p3d.build_layout(SHAPE, (4, 4, 4), radius=1, pool_size=1, layout="raster_block", device=gpu)
    layer = _layers("axial", p3d.RotaryEncoding("half", 0.5))[0].to(gpu, torch.bfloat16).eval()
    xs = [torch.randn(1, math.prod(SHAPE), DIM, device=gpu).bfloat16() for _ in range(3)]
    gate = torch.rand(1, 1, DIM, device=gpu).bfloat16()

    def step(x):
        return layer(x, lay, residual_gate=gate, next_norm=p3d.Norm("rms"))
    with torch.inference_mode():
        eager = [step(x) for x in xs]
        held = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(held)
        for i in (0, 1, 2, 0):
            held.copy_(xs[i])
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, eager[i]):
                assert torch.equal(a, b), i
            step(xs[1])
            torch.cuda.synchronize()


def test_layer_refusals(gpu):
    lay = p3d.build_layout(SHAPE, (4, 4, 4), radius=1, pool_size=1, layout="raster_block", device=gpu)
    layer = p3d.PACK3DAttention(DIM, heads=HEADS, kv_heads=KV, head_dim=HEAD_DIM, block_volume=64).to(gpu)
    x = torch.randn(1, math.prod(SHAPE), DIM, device=gpu)
    for kw in ({"normed": x[:, :1]}, {"next_norm": torch.nn.Linear(2, 2)}, {"next_norm": p3d.Norm("other")},
               {"residual_gate": x[:, :3]}, {"residual_gate": x[0]}):
        with pytest.raises(ValueError):
            layer(x, lay, **kw)
    turned = p3d.PACK3DAttention(DIM, heads=HEADS, kv_heads=KV, head_dim=HEAD_DIM, block_volume=64,
                                 rotary=p3d.RotaryEncoding()).to(gpu)
    with pytest.raises(ValueError, match="RotaryEncoding"):
        turned.core_inputs(x, lay)


@pytest.mark.parametrize("kw", [{"y": 1}, {"gate": 1}, {"gate": 2}, {"scale": 1}, {"post_norm": 1}, {"post_norm": 2}, {"alpha": float("inf")},
                                {"p": 1.0, "seed": 1}, {"p": 0.5}, {"next_norm": 3}])
def test_residual_refusals(gpu, kw):
    x = torch.randn(2, 5, 24, device=gpu)
    bad = {"y": {1: x[:, :4]}, "gate": {1: x[:1], 2: x.double()}, "scale": {1: torch.ones(23, device=gpu)},
           "post_norm": {1: p3d.Norm("rms", torch.ones(25, device=gpu)), 2: p3d.Norm("rms", None, torch.ones(24))},
           "next_norm": {3: p3d.Norm("layer", eps=-1.0)}}
    kw = {k: bad[k][v] if k in bad else v for k, v in kw.items()}
    y = kw.pop("y", x)
    with pytest.raises(ValueError):
        p3d.block_residual(x, y, **kw)


def test_type_refusals(gpu):
    x = torch.randn(2, 5, 24, device=gpu)
    for a, b in ((x.half(), x), (x.bfloat16(), x.half()), (x.double(), x), (x, x.double())):
        with pytest.raises(ValueError):
            p3d.block_residual(a, b)
    for a, dt in ((x.half(), torch.float32), (x.half(), torch.bfloat16), (x, torch.float64)):
        with pytest.raises(ValueError):
            p3d.block_norm(a, p3d.Norm(), dtype=dt)
    for a in (torch.empty(2, 5, 8193, device=gpu), x[0, 0], x[None], torch.empty(2, 5, 0, device=gpu)):
        with pytest.raises(ValueError):
            p3d.block_norm(a, p3d.Norm())
    with pytest.raises(ValueError):
        p3d.block_norm(x, None)
    with pytest.raises(ValueError):
        p3d.counter_dropout(x.double(), 0.5, 1)


def test_rotary_refusals(gpu):
    q = torch.randn(2, 4, 6, 16, device=gpu)
    pos, freqs = torch.arange(6, device=gpu), p3d.rotary_frequencies(8)[0].to(gpu)
    good = {"tensors": q, "positions": pos, "freqs": freqs}
    p3d.apply_rotary(**good)
    for change in ({"tensors": q[0]}, {"tensors": (q, q[:, :, :5])}, {"tensors": (q, q.half())}, {"tensors": ()}, {"tensors": [q] * 5},
                   {"tensors": q.double()}, {"positions": pos[:5]}, {"positions": pos.float()}, {"positions": pos.cpu()},
                   {"positions": pos.expand(3, 6)}, {"freqs": freqs.float()}, {"freqs": freqs.cpu()},
                   {"freqs": p3d.rotary_frequencies(9)[0].to(gpu)}, {"pairs": (4, 5)}, {"pairs": (4, 4)}, {"pairs": (2, 2, 2, 2)},
                   {"layout": "other"}, {"magnitude": float("nan")}, {"tensors": q[:, :0]},
                   {"tensors": torch.randn(1, 3000, 1, 16, device=gpu), "positions": pos[:1]}):
        with pytest.raises(ValueError):
            p3d.apply_rotary(**{**good, **change})
