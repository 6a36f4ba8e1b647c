"""block_norm and block_residual against their definition in 64 bits: outputs, every
gradient, the kinds of gates, widths from 1 to 8192, strides, empty inputs, values that
are not finite, a captured graph, another stream."""
import pytest
import torch

import pack3d_amd as p3d
from tests._block_reference import (assert_within, block_reference, half_step, keep_mask, keep_mask_at, smallest,
                                    sum_bound)

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(gen, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype)


def _case(gpu, batch, tokens, dim, outer, inner, post, after, gate, scale, alpha, p, param=None, seed=0, grads=True):
    """Inputs of one call on the device, and what the definition gives for them."""
    gen = torch.Generator().manual_seed(seed + dim * 31 + tokens)
    param = param or (inner if outer == inner else F32)
    rows = batch * tokens
    t = {"x": _rand(gen, batch, tokens, dim, dtype=outer, std=1.5, mean=0.2), "y": _rand(gen, batch, tokens, dim, dtype=inner)}
    for name, kind in (("", post), ("next_", after)):
        if kind:
            t[name + "weight"] = _rand(gen, dim, dtype=param, std=0.1, mean=1.0)
            if kind == "layer":
                t[name + "bias"] = _rand(gen, dim, dtype=param, std=0.1)
    shape = {"sample": (batch, 1, dim), "shared": (1, 1, dim), "token": (batch, tokens, 1), "full": (batch, tokens, dim)}
    if gate:
        t["gate"] = _rand(gen, *shape[gate], dtype=inner, std=0.4, mean=0.5)
    if scale:
        t["scale"] = _rand(gen, dim, dtype=param, std=0.2, mean=0.5)
    up = {"out": _rand(gen, batch, tokens, dim, dtype=outer)}
    if after:
        up["n"] = _rand(gen, batch, tokens, dim, dtype=inner)
    seeds = (0x1234567890ABCDEF + seed, 5 + seed)
    threshold = int(p * 65536 + 0.5)

    def wide(name):
        return None if name not in t else t[name].double()

    def norm(kind, pre):
        return (kind, wide(pre + "weight"), wide(pre + "bias"), 1e-5) if kind else None
    g = None if not gate else t["gate"].double().expand(batch, tokens, dim).reshape(rows, dim)
    keep = keep_mask(rows * dim, threshold, *seeds).view(rows, dim) if p else None
    ref = block_reference(wide("x").view(rows, dim), wide("y").view(rows, dim), norm(post, ""), g, wide("scale"), alpha,
                          keep, threshold / 65536, norm(after, "next_"),
                          up["out"].double().view(rows, dim) if grads else None,
                          up["n"].double().view(rows, dim) if grads and after else None)
    if grads and gate:
        terms, dterms = (v.view(batch, tokens, dim) for v in ref.pop("d_gate_terms"))
        axes = [i for i, (a, b) in enumerate(zip(shape[gate], (batch, tokens, dim))) if a != b]
        if axes:
            bound = sum_bound(terms, dterms, rows * (1 if axes[0] < 2 else 0) + dim * (axes[-1] == 2), axes).reshape(shape[gate])
            ref["d_gate"] = (terms.sum(axes, keepdim=True), bound)
        else:
            ref["d_gate"] = (terms, dterms)
    dev = {k: v.to(gpu) for k, v in t.items()}
    upd = {k: v.to(gpu) for k, v in up.items()}
    return dev, upd, ref, seeds


def _call(dev, post, after, alpha, p, seeds):
    def norm(kind, pre):
        return p3d.Norm(kind, dev[pre + "weight"], dev.get(pre + "bias"), 1e-5) if kind else None
    got = p3d.block_residual(dev["x"], dev["y"], post_norm=norm(post, ""), gate=dev.get("gate"), scale=dev.get("scale"),
                             alpha=alpha, p=p, seed=seeds, next_norm=norm(after, "next_"))
    return {"out": got[0], "n": got[1]} if after else {"out": got}


def _check(name, got, ref):
    value, bound = ref
    assert_within(got.reshape(value.shape), value,
                  bound + (half_step(got.dtype) * (value.abs() + bound) + smallest(got.dtype)), name)


def _run_case(gpu, post, after, alpha, p, *args, **kw):
    batch, tokens, dim, outer, inner, gate, scale = args
    dev, up, ref, seeds = _case(gpu, batch, tokens, dim, outer, inner, post, after, gate, scale, alpha, p, **kw)
    with torch.no_grad():
        plain = _call(dev, post, after, alpha, p, seeds)
    for t in dev.values():
        t.requires_grad_()
    outs = _call(dev, post, after, alpha, p, seeds)
    for k in outs:
        assert torch.equal(outs[k], plain[k]), k  # with and without a graph
        _check(k, outs[k], ref[k])
    grads = torch.autograd.grad(list(outs.values()), list(dev.values()), [up[k] for k in outs])
    for name, g in zip(dev, grads):
        assert g.dtype == dev[name].dtype and g.shape == dev[name].shape
        _check("d_" + name, g, ref["d_" + name])


TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]


@pytest.mark.parametrize("outer,inner", TYPES)
@pytest.mark.parametrize("post,after,gate,scale,alpha,p", [
    (None, None, None, False, 1.0, 0.0),
    ("layer", "layer", "sample", True, 1.0, 0.1),
    ("rms", "rms", "token", True, 1.5, 0.0),
    ("rms", None, "full", False, 1.0, 0.3),
    (None, "layer", "full", True, 0.5, 0.1),
    ("layer", None, "token", False, 1.0, 0.25),
    (None, "rms", "sample", False, 1.0, 0.0),
    ("layer", "rms", "shared", True, 2.0, 0.5),
    (None, None, "sample", True, 1.0, 0.1),
])
def test_residual_kinds(gpu, outer, inner, post, after, gate, scale, alpha, p):
    _run_case(gpu, post, after, alpha, p, 3, 37, 72, outer, inner, gate, scale)


@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 32, 33, 63, 64, 65, 96, 97, 128, 131, 160, 192, 200, 256, 264, 327,
                                 384, 385, 512, 513, 520, 768, 769, 1000, 1024, 1025, 1500, 1536, 1537, 2048, 2049, 2560, 2561, 3001, 3584,
                                 3585, 4096, 4097, 5001, 8191, 8192])
def test_residual_widths(gpu, dim):
    print(f"block_residual dim {dim}", flush=True)
    _run_case(gpu, "layer", "rms", 1.25, 0.1, 2, 5, dim, F32, BF16, "sample", True)
    _run_case(gpu, "layer", "layer", 1.0, 0.3, 1, 70, dim, F32, F32, "full", True)
    _run_case(gpu, "rms", "layer", 1.0, 0.2, 1, 3, dim, F16, F16, "token", True)


@pytest.mark.parametrize("batch,tokens", [(1, 1), (1, 2), (7, 1), (1, 999), (600, 3), (5000, 1), (2, 4099), (1, 40000)])
def test_residual_rows(gpu, batch, tokens):
    _run_case(gpu, "rms", "layer", 1.0, 0.1, batch, tokens, 40, F32, BF16, "sample", True)
    _run_case(gpu, None, None, 1.0, 0.0, batch, tokens, 40, BF16, BF16, "sample", False)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("outer,inner", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 4096), (3, 1), (300, 192), (77, 515), (4000, 64), (9, 8192)])
def test_block_norm(gpu, kind, outer, inner, rows, dim):
    gen = torch.Generator().manual_seed(rows + dim)
    x = _rand(gen, rows, dim, dtype=outer, std=2.0, mean=1.0)
    w, b = _rand(gen, dim, std=0.1, mean=1.0), _rand(gen, dim, std=0.1)
    dn = _rand(gen, rows, dim, dtype=inner)
    ref = block_reference(x.double(), None, None, None, None, 1.0, None, 0.0, (kind, w.double(), b.double(), 1e-6), None,
                          dn.double())
    x, w, b = (t.to(gpu).requires_grad_() for t in (x, w, b))
    n = p3d.block_norm(x, p3d.Norm(kind, w, b, 1e-6), dtype=inner)
    assert n.dtype == inner
    _check("n", n, ref["n"])
    for name, g in zip(("d_x", "d_next_weight", "d_next_bias"), torch.autograd.grad(n, (x, w, b), dn.to(gpu))):
        _check(name, g, ref[name])


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_block_norm_without_affine_and_from_modules(gpu, kind):
    gen = torch.Generator().manual_seed(3)
    x = _rand(gen, 2, 50, 96, dtype=BF16).to(gpu).requires_grad_()
    dn = _rand(gen, 2, 50, 96, dtype=BF16).to(gpu)
    ref = block_reference(x.detach().double().cpu().view(100, 96), None, None, None, None, 1.0, None, 0.0,
                          (kind, None, None, 1e-5), None, dn.double().cpu().view(100, 96))
    n = p3d.block_norm(x, p3d.Norm(kind))
    _check("n", n, ref["n"])
    _check("d_x", torch.autograd.grad(n, x, dn)[0], ref["d_x"])
    module = (torch.nn.LayerNorm(96) if kind == "layer" else torch.nn.RMSNorm(96, eps=1e-5)).to(gpu)
    assert torch.equal(p3d.block_norm(x, p3d.Norm.of(module)), n)


def test_a_full_step_agrees_with_differences(gpu):
    """The gradients of fp32 inputs against central differences of the definition in 64 bits along
    random directions: a difference of step 1e-5 is off by its third derivative times 1e-10, far
    below the 1e-4 of the sum that the gradients' fp32 rounding is allowed."""
    dev, up, ref, seeds = _case(gpu, 2, 9, 24, F32, F32, "layer", "rms", "sample", True, 1.5, 0.2, grads=True)
    for t in dev.values():
        t.requires_grad_()
    outs = _call(dev, "layer", "rms", 1.5, 0.2, seeds)
    grads = dict(zip(dev, torch.autograd.grad(list(outs.values()), list(dev.values()), [up[k] for k in outs])))
    base = {k: v.detach().double().cpu() for k, v in dev.items()}
    keep = keep_mask(18 * 24, int(0.2 * 65536 + 0.5), *seeds).view(18, 24)

    def loss(t):
        made = block_reference(t["x"].view(18, 24), t["y"].view(18, 24), ("layer", t["weight"], t["bias"], 1e-5),
                               t["gate"].expand(2, 9, 24).reshape(18, 24), t["scale"], 1.5, keep,
                               int(0.2 * 65536 + 0.5) / 65536, ("rms", t["next_weight"], None, 1e-5), None, None)
        return sum((made[k][0] * up[k].double().cpu().view(18, 24)).sum() for k in ("out", "n"))
    gen = torch.Generator().manual_seed(8)
    for name in base:
        step = torch.randn(base[name].shape, generator=gen, dtype=torch.float64)
        plus, minus = ({**base, name: base[name] + s * 1e-5 * step} for s in (1, -1))
        difference = (loss(plus) - loss(minus)) / 2e-5
        terms = grads[name].double().cpu() * step
        assert abs(terms.sum() - difference) <= 1e-4 * terms.abs().sum(), name


def test_strided_inputs_and_upstream(gpu):
    """Rows of a wider buffer, channels at odd offsets, expanded rows and expanded gradients: the same bits as
    contiguous copies."""
    gen = torch.Generator().manual_seed(4)
    wide = _rand(gen, 2, 33, 3 * 50 + 1, dtype=BF16).to(gpu)
    x, y, gate = wide[..., 1:51], wide[..., 51:101], wide[..., 101:]
    w = _rand(gen, 50, dtype=BF16, mean=1.0).to(gpu)

    def run(x, y, gate, transposed=False):
        x, y, gate = (t.detach().requires_grad_() for t in (x, y, gate))
        out, n = p3d.block_residual(x, y, post_norm=p3d.Norm("rms", w), gate=gate, p=0.1, seed=3,
                                    next_norm=p3d.Norm("layer"))
        return (out, n, *torch.autograd.grad((out, n), (x, y, gate), (torch.ones_like(out) if not transposed else
                                                                     torch.ones((), dtype=BF16, device=gpu).expand_as(out),
                                                                     wide[..., 7:57])))
    for a, b in zip(run(x, y, gate, True), run(*(t.contiguous() for t in (x, y, gate)))):
        assert torch.equal(a, b)
    # channels not contiguous, rows expanded
    xt = _rand(gen, 50, 33, dtype=BF16).to(gpu).t().expand(2, 33, 50)
    row = y[:, :1].expand(2, 33, 50)
    for a, b in zip(run(xt, row, gate), run(xt.contiguous(), row.contiguous(), gate)):
        assert torch.equal(a, b)


def test_rows_that_are_not_finite_stay_by_themselves(gpu):
    """An infinity or NaN shows in its own row of out and n and in no other row, and one that the mask drops
    does not show at all."""
    gen = torch.Generator().manual_seed(5)
    x, y = (_rand(gen, 1, 40, 72).to(gpu) for _ in range(2))
    clean = p3d.block_residual(x, y, post_norm=p3d.Norm("rms"), next_norm=p3d.Norm("layer"))
    for value in (float("inf"), float("nan")):
        bad = y.clone()
        bad[0, 13, 70] = value
        got = p3d.block_residual(x, bad, post_norm=p3d.Norm("rms"), next_norm=p3d.Norm("layer"))
        others = [i for i in range(40) if i != 13]
        for a, b in zip(got, clean):
            assert torch.equal(a[0, others], b[0, others])
            assert not torch.isfinite(a[0, 13]).all()
    keep = keep_mask(40 * 72, 32768, 9, 0).view(40, 72)
    bad = torch.where(keep.to(gpu), y[0], float("nan"))[None].requires_grad_()
    out = p3d.block_residual(x, bad, p=0.5, seed=9)
    assert torch.isfinite(out).all()
    (dy,) = torch.autograd.grad(out, bad, torch.ones_like(out))
    assert torch.equal(dy[0] != 0, keep.to(gpu))


def test_empty_inputs(gpu):
    for shape in ((0, 5, 24), (2, 0, 24), (0, 24)):
        x, y = (torch.zeros(shape, device=gpu, requires_grad=True) for _ in range(2))
        w = torch.ones(24, device=gpu, requires_grad=True)
        out, n = p3d.block_residual(x, y, post_norm=p3d.Norm("rms", w), next_norm=p3d.Norm("layer", w))
        grads = torch.autograd.grad((out, n), (x, y, w), (out, n))
        assert out.shape == n.shape == shape and grads[0].shape == shape and not grads[2].any()


def test_only_what_is_needed(gpu):
    """Gradients that nothing asks for are None, and an output that nothing uses counts as zero."""
    gen = torch.Generator().manual_seed(6)
    x, y = (_rand(gen, 2, 20, 48).to(gpu).requires_grad_() for _ in range(2))
    w = (_rand(gen, 48).to(gpu) + 1).requires_grad_()
    gate = _rand(gen, 2, 1, 48).to(gpu)
    up = _rand(gen, 2, 20, 48).to(gpu)

    def run():
        return p3d.block_residual(x, y, post_norm=p3d.Norm("rms", w), gate=gate, next_norm=p3d.Norm("layer", w))
    out, n = run()
    only_n = torch.autograd.grad(n, (x, y, w), up)
    out, n = run()
    both = torch.autograd.grad((out, n), (x, y, w), (torch.zeros_like(out), up))
    for a, b in zip(only_n, both):
        assert torch.equal(a, b)
    out, n = run()
    dx, dw = torch.autograd.grad(out, (x, w), up)
    assert torch.equal(dx, up)
    plain = p3d.block_residual(x, y, post_norm=p3d.Norm("rms", w), gate=gate)
    assert torch.equal(torch.autograd.grad(plain, w, up)[0], dw)
    frozen = p3d.block_residual(x.detach(), y.detach(), post_norm=p3d.Norm("rms", w), gate=gate)
    assert torch.equal(torch.autograd.grad(frozen, w, up)[0], dw)


def test_repeats_bit_for_bit_and_on_another_stream(gpu):
    def run():
        dev, up, _, seeds = _case(gpu, 3, 700, 192, F32, BF16, "rms", "layer", "sample", True, 1.0, 0.1, grads=False)
        for t in dev.values():
            t.requires_grad_()
        outs = _call(dev, "rms", "layer", 1.0, 0.1, seeds)
        return (*outs.values(), *torch.autograd.grad(list(outs.values()), list(dev.values()), [up[k] for k in outs]))
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_training_step_in_a_graph(gpu):
    """Forward and backward captured once and replayed on new inputs and new seeds, against eager calls."""
    gen = torch.Generator().manual_seed(7)
    shape = (2, 65, 80)
    sets = [[_rand(gen, *shape).to(gpu) for _ in range(3)] for _ in range(3)]
    seeds = [torch.tensor([11 + i, i], device=gpu) for i in range(3)]
    w0 = _rand(gen, 80, mean=1.0).to(gpu)

    def step(x, y, up, seed):
        x, y, w = (t.detach().requires_grad_() for t in (x, y, w0))
        gate = torch.full((2, 1, 80), 0.5, device=gpu, requires_grad=True)
        out, n = p3d.block_residual(x, y, post_norm=p3d.Norm("rms", w), gate=gate, p=0.2, seed=seed,
                                    next_norm=p3d.Norm("layer"))
        return (out.detach(), n.detach(), *torch.autograd.grad((out, n), (x, y, w, gate), (up, up)))
    eager = [step(*s, seed) for s, seed in zip(sets, seeds)]
    held = [t.clone() for t in sets[0]]
    held_seed = seeds[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held, held_seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held, held_seed)
    for i in (0, 1, 2, 0):
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        held_seed.copy_(seeds[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, eager[i]):
            assert torch.equal(a, b), i
        step(*sets[1], seeds[1])
        torch.cuda.synchronize()


def test_first_step_of_its_kind_in_a_graph(gpu):
    """A width and gate that nothing ran before, captured at once."""
    x, y, gate, up = (torch.randn(300, 1001, device=gpu).half() for _ in range(4))

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, y, gate)]
        out = p3d.block_residual(leaves[0], leaves[1], gate=leaves[2], p=0.25, seed=5, alpha=0.5)
        return (out.detach(), *torch.autograd.grad(out, leaves, up))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    want = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
            a.zero_()


@pytest.mark.parametrize("way", ["norm", "residual", "dropout", "rotary"])
def test_captured_backward_while_an_eager_graph_lives(gpu, way):
    """Refused while an eager graph of the leaf on the default stream is alive, and right once it is dropped."""
    freqs, positions = p3d.rotary_frequencies(8)[0].to(gpu), torch.arange(6, device=gpu)
    call = {"norm": lambda x: p3d.block_norm(x, p3d.Norm("rms")),
            "residual": lambda x: p3d.block_residual(x, x.detach() * 2, p=0.3, seed=4, alpha=2.0),
            "dropout": lambda x: p3d.counter_dropout(x, 0.3, 4),
            "rotary": lambda x: p3d.apply_rotary(x, positions, freqs)}[way]
    x = torch.randn(1, 2, 6, 16, device=gpu) if way == "rotary" else torch.randn(2, 6, 16, device=gpu)
    x.requires_grad_()
    up = torch.randn_like(x)
    want, = torch.autograd.grad(call(x), x, up)
    alive = call(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured into a graph while an eager graph"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(call(x), x, up)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(call(x), x, up)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_inputs_changed_before_the_backward_raise(gpu):
    x, y = (torch.randn(1, 4, 16, device=gpu, requires_grad=True) for _ in range(2))
    seed = torch.tensor([1, 2], device=gpu)
    out = p3d.block_residual(x, y, p=0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out.sum(), x)


def _ways(gpu):
    """One call of each operator on a leaf x: name -> (leaf, function of it)."""
    freqs = p3d.rotary_frequencies(8)[0].to(gpu)
    positions = torch.arange(6, device=gpu)
    w = torch.ones(24, device=gpu, requires_grad=True)
    gate = torch.full((2, 1, 24), 0.5, device=gpu)

    def leaf(*shape):
        return torch.randn(*shape, device=gpu, requires_grad=True)
    return {"residual": (leaf(2, 5, 24), lambda x: p3d.block_residual(x, x.detach() * 2, post_norm=p3d.Norm("rms", w), gate=gate,
                                                                       p=0.3, seed=4, next_norm=p3d.Norm("layer", w))[1]),
            "norm": (leaf(7, 24), lambda x: p3d.block_norm(x, p3d.Norm("layer", w))),
            "dropout": (leaf(7, 24), lambda x: p3d.counter_dropout(x, 0.3, 4)),
            "rotary": (leaf(2, 3, 6, 16), lambda x: p3d.apply_rotary(x, positions, freqs))}


@pytest.mark.parametrize("name", ["residual", "norm", "dropout", "rotary"])
def test_autograd_contract(gpu, name):
    """A graph kept and gone, saved tensors that come back as others, second order and forward mode refused."""
    x, f = _ways(gpu)[name]
    up = torch.randn_like(f(x))
    (g,) = torch.autograd.grad(f(x), x, up)
    out = f(x)
    assert torch.equal(torch.autograd.grad(out, x, up, retain_graph=True)[0], g)
    assert torch.equal(torch.autograd.grad(out, x, up)[0], g)
    if name in ("residual", "norm", "rotary"):
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(out, x, up)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(gpu)):
        moved = f(x)
    assert torch.equal(torch.autograd.grad(moved, x, up)[0], g)
    again = up.clone().requires_grad_()
    (first,) = torch.autograd.grad(f(x), x, again, create_graph=True)
    assert torch.equal(first.detach(), g) and first.requires_grad
    for by in (again, x) if name in ("residual", "norm") else (again,):  # the others are linear in x
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(first.sum(), by, retain_graph=True)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        dual = fwad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(dual)
    x.grad = None
    f(x).backward(up)
    f(x).backward(up)
    assert torch.allclose(x.grad, 2 * g)


def test_calls_from_two_threads(gpu):
    """Each thread on a stream of its own, forward and backward, against the same calls made alone."""
    import threading
    shapes = [(2, 300, 192), (1, 700, 327)]

    def work(shape, seed):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        x, y, up = (torch.randn(shape, generator=gen, device=gpu) for _ in range(3))
        x, y = x.requires_grad_(), y.requires_grad_()
        out, n = p3d.block_residual(x, y, post_norm=p3d.Norm("rms"), p=0.2, seed=seed, next_norm=p3d.Norm("layer"))
        return [out.detach(), n.detach(), *torch.autograd.grad((out, n), (x, y), (up, up))]
    alone = [work(s, i) for i, s in enumerate(shapes)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = work(shapes[i], i)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, got):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_rows_beyond_four_gigabytes(gpu):
    """Rows 8 MiB apart (their last bytes past 2^33) read as contiguous copies of them do."""
    rows, stride = 1100, 1 << 22
    big = torch.empty(rows * stride, dtype=BF16, device=gpu)
    x, y, gate, up = (big.as_strided((rows, 72), (stride, 1), 512 * i) for i in range(4))
    gen = torch.Generator(device=gpu).manual_seed(1)
    for t in (x, y, gate, up):
        t.copy_(torch.randn(rows, 72, generator=gen, device=gpu))

    def run(x, y, gate, up):
        x, y, gate = (t.detach().requires_grad_() for t in (x, y, gate))
        out, n = p3d.block_residual(x, y, post_norm=p3d.Norm("layer"), gate=gate, p=0.1, seed=5, next_norm=p3d.Norm("rms"))
        return (out, n, *torch.autograd.grad((out, n), (x, y, gate), (up, up)))
    for a, b in zip(run(x, y, gate, up), run(*(t.contiguous() for t in (x, y, gate, up)))):
        assert torch.equal(a, b)
    far = big.as_strided((5, 64), (1 << 29, 1))  # a stride that is copied before the kernel
    far.copy_(torch.randn(5, 64, device=gpu))
    assert torch.equal(p3d.block_norm(far, p3d.Norm("rms")), p3d.block_norm(far.contiguous(), p3d.Norm("rms")))


def test_outputs_beyond_four_gigabytes(gpu):
    """2^31 and some elements: the last rows of each output as a call on those rows alone gives them."""
    rows, dim = 33_600_000, 64
    x = torch.empty(rows, dim, dtype=BF16, device=gpu)
    x.normal_()
    n = p3d.block_norm(x, p3d.Norm("layer"))
    assert torch.equal(n[-100:], p3d.block_norm(x[-100:], p3d.Norm("layer")))
    del n
    y = p3d.counter_dropout(x, 0.25, (3, 4))
    first = (rows - 2) * dim
    keep = keep_mask_at(first, 2 * dim, 16384, 3, 4)
    inv = torch.tensor(65536.0 / 49152.0, dtype=F32)
    assert torch.equal(y[-2:].cpu().flatten(), torch.where(keep, x[-2:].cpu().flatten().float() * inv, 0.0).to(BF16))
    out = p3d.block_residual(torch.zeros_like(x), x, p=0.25, seed=(3, 4))
    assert torch.equal(out[-2:], y[-2:])
