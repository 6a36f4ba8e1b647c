"""Operators around the PACK3D attention block: what is measured of them.

* ``norm``    -- the norm before a block (``block_norm``),
* ``close``   -- the end of a block (``block_residual``): the norm after it, dropout,
  its gate, the residual scale, the sum and the next block's norm,
* ``rotary``  -- rotary positions of queries and keys (``apply_rotary``),
* ``dropout`` -- dropout from a counter-based generator (``counter_dropout``).

``infer`` is the forward pass alone, ``train`` the forward pass and the gradients
of every floating input.  Tensors are [batch, tokens, dim], heads [batch, heads,
tokens, head_dim] as views of the projections.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
# (type of the residual stream, type inside the block)
TYPES = {"fp32": (torch.float32, torch.float32), "fp16": (torch.float16, torch.float16),
         "bf16": (torch.bfloat16, torch.bfloat16), "mixed": (torch.float32, torch.bfloat16)}


def _norm_case(name, way, batch, tokens, dim, kind, dtype, affine="weight_bias"):
    case = {"op": "norm", "way": way, "batch": batch, "tokens": tokens, "dim": dim, "kind": kind, "dtype": dtype,
            "affine": affine}
    return dict(case, name=name) if name else case


def _close_case(name, way, batch, tokens, dim, post, after, dtype, *, gate="none", scale=False, p=0.0, alpha=1.0):
    case = {"op": "close", "way": way, "batch": batch, "tokens": tokens, "dim": dim, "post": post, "next": after,
            "dtype": dtype, "gate": gate, "scale": scale, "p": p, "alpha": alpha}
    return dict(case, name=name) if name else case


def _rotary_case(name, way, batch, tokens, heads, kv_heads, keys, head_dim, pairs, axes, layout, scaling, far, dtype):
    case = {"op": "rotary", "way": way, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "keys": keys, "head_dim": head_dim, "pairs": pairs, "axes": axes, "layout": layout, "scaling": scaling,
            "far": far, "dtype": dtype}
    return dict(case, name=name) if name else case


def _dropout_case(name, way, batch, tokens, dim, p, dtype):
    case = {"op": "dropout", "way": way, "batch": batch, "tokens": tokens, "dim": dim, "p": p, "dtype": dtype}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token of a wide model's served sequence: the call's latency.
        _norm_case("norm_token", "infer", 1, 1, 4096, "rms", "bf16", "weight"),
        # The first norm of a training step under autocast: fp32 stream, bf16 out, 16 x 64 x 64 voxels.
        _norm_case("norm_train", "train", 1, 65536, 512, "layer", "mixed"),
        # The end of a block for one token, with the next block's norm.
        _close_case("close_token", "infer", 1, 1, 512, "rms", "rms", "bf16", gate="sample"),
        # The end of a block of a 64^3 volume that a conditioned model is served on.
        _close_case("close_volume", "infer", 1, 262144, 192, "none", "layer", "bf16", gate="sample", scale=True),
        # The whole end of a block in training, on the same volume under autocast.
        _close_case("close_train", "train", 1, 262144, 192, "rms", "layer", "mixed", gate="sample", scale=True,
                    p=0.1),
        # Three 17^3 volumes, an odd width, a gate of its own for each element, fp16, a scaled residual.
        _close_case("close_ragged", "train", 3, 4913, 327, "layer", "none", "fp16", gate="full", p=0.25, alpha=2.0),
        # A wide model's block: two sequences, one gate value a token.
        _close_case("close_wide", "train", 2, 4096, 4096, "rms", "rms", "bf16", gate="token"),
        # One new token for each of eight sequences, far out: half layout, whole heads.
        _rotary_case("rotary_token", "infer", 8, 1, 8, 2, 1, 64, 32, 1, "half", "ntk", 1000000, "bf16"),
        # The rotation of q, kl and kg of a 64^3 volume by its coordinates, on a grid larger than trained on.
        _rotary_case("rotary_volume", "infer", 1, 262144, 4, 4, 2, 48, 24, 3, "interleaved", "linear", 0, "bf16"),
        # Training in fp32 on two ragged sequences, half of each head rotated, frequencies scaled by parts.
        _rotary_case("rotary_train", "train", 2, 18711, 8, 2, 1, 128, 32, 1, "half", "parts", 5000, "fp32"),
        # Dropout of a 16^3 volume of a small model.
        _dropout_case("dropout_small", "infer", 1, 4096, 64, 0.1, "bf16"),
        # Dropout in training on a 64^3 volume of a wide layer.
        _dropout_case("dropout_train", "train", 1, 262144, 512, 0.1, "bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _dim(rng, low=16, high=4096):
    """A width: a multiple of 8 more often than not, as models have them, else as it comes."""
    dim = _log(rng, low, high)
    return max(low, dim // 8 * 8) if rng.random() < 0.6 else dim


def _tokens(rng, dim, batch, most):
    return max(1, min(_log(rng, 1, 262144), most // (dim * batch)))


def draw(rng):
    op = rng.choice(["norm", "close", "close", "rotary", "dropout"])
    way = rng.choice(["infer", "train"])
    dtype = rng.choice(list(TYPES))
    batch = rng.choice([1, 1, 2, 3, 5, 8])
    if op == "norm":
        dim = _dim(rng)
        return _norm_case(None, way, batch, _tokens(rng, dim, batch, 33_000_000), dim, rng.choice(["layer", "rms"]),
                          dtype, rng.choice(["weight_bias", "weight", "none"]))
    if op == "close":
        dim = _dim(rng)
        return _close_case(None, way, batch, _tokens(rng, dim, batch, 40_000_000), dim,
                           rng.choice(["none", "layer", "rms"]), rng.choice(["none", "layer", "rms"]), dtype,
                           gate=rng.choice(["none", "sample", "token", "full"]), scale=rng.random() < 0.5,
                           p=rng.choice([0.0, 0.05, 0.1, 0.3]), alpha=rng.choice([1.0, 1.0, 1.5]))
    dtype = "bf16" if dtype == "mixed" else dtype
    if op == "dropout":
        dim = _dim(rng)
        return _dropout_case(None, way, batch, _tokens(rng, dim, batch, 100_000_000), dim,
                             rng.choice([0.05, 0.1, 0.3, 0.5]), dtype)
    kv_heads = rng.choice([1, 2, 4])
    heads = kv_heads * rng.choice([1, 2, 4])
    head_dim = rng.choice([16, 32, 48, 64, 80, 128])
    axes = rng.choice([1, 1, 3])
    pairs = max(3, head_dim // 2 if rng.random() < 0.5 else rng.randint(3, head_dim // 2))
    keys = rng.choice([1, 2])
    tokens = _tokens(rng, head_dim * (heads + keys * kv_heads), batch, 40_000_000)
    return _rotary_case(None, way, batch, tokens, heads, kv_heads, keys, head_dim, pairs, axes,
                        rng.choice(["interleaved", "half"]), rng.choice(["none", "linear", "ntk", "parts"]),
                        0 if axes == 3 else _log(rng, 1, 1000000), dtype)


def _axis_pairs(case):
    """How many of the rotary pairs each axis has, the remainder first."""
    pairs, axes = case["pairs"], case["axes"]
    return tuple(pairs // axes + (a < pairs % axes) for a in range(axes))


def _frequencies(count, scaling, factor=4.0, trained=8192.0, base=10000.0):
    """Radians a position of one axis' pairs, in 64 bits, and the factor on rotated channels: as trained,
    positions interpolated, the base raised, or interpolated by how often a pair turns over the trained length."""
    j = torch.arange(count, dtype=torch.float64)
    freq, magnitude = base ** (-j / count), 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ntk":
        freq = (base * factor ** (count / max(1, count - 1))) ** (-j / count)
    elif scaling == "parts":
        kept = ((trained * freq / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freq = freq * kept + freq / factor * (1.0 - kept)
        magnitude = 0.1 * math.log(factor) + 1.0
    return freq, magnitude


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 17)
    grad = case["way"] == "train"
    outer, inner = TYPES[case["dtype"]]
    b, n = case["batch"], case["tokens"]

    def normal(*shape, dtype=inner, mean=0.0, std=1.0, leaf=True):
        t = torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).mul_(std).add_(mean).to(dtype)
        return t.requires_grad_(grad and leaf)

    def key():
        return torch.randint(0, 2 ** 62, (2,), generator=gen, device=DEVICE, dtype=torch.int64)

    s = {"case": dict(case)}
    if case["op"] == "dropout":
        s["x"], s["key"] = normal(b, n, case["dim"]), key()
        if grad:
            s["dy"] = normal(b, n, case["dim"], leaf=False)
        return s
    if case["op"] == "rotary":
        h, g, d, keys = case["heads"], case["kv_heads"], case["head_dim"], case["keys"]
        qp = normal(b, n, h * d, leaf=False)
        kp = normal(b, n, 2 * keys * g * d, leaf=False)  # keys and values, in chunks
        heads = [qp.view(b, n, h, d).transpose(1, 2)]
        heads += [t.transpose(1, 2) for t in kp.view(b, n, 2 * keys, g, d).unbind(2)[::2]]
        s["heads"] = [t.detach().requires_grad_(grad) for t in heads]
        if case["axes"] == 3:
            side = max(1, round(n ** (1 / 3)))
            i = torch.arange(n, device=DEVICE)
            s["positions"] = torch.stack((i // (side * side), i // side % side, i % side), -1)
        else:
            first = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device=DEVICE)
            s["positions"] = first + torch.arange(n, device=DEVICE)
        made = [_frequencies(count, case["scaling"]) for count in _axis_pairs(case)]
        s["freqs"], s["magnitude"] = torch.cat([f for f, _ in made]).to(DEVICE), made[0][1]
        if grad:
            s["douts"] = [normal(b, t.shape[1], n, d, leaf=False) for t in heads]
        return s
    dim = case["dim"]
    half = outer != torch.float32
    param = inner if half else torch.float32

    def affine(kind, which="weight_bias"):
        w = normal(dim, dtype=param, mean=1.0, std=0.1) if kind != "none" and "weight" in which else None
        return w, normal(dim, dtype=param, std=0.1) if kind != "none" and "bias" in which else None

    s["x"] = normal(b, n, dim, dtype=outer, mean=0.1, std=1.5)
    if case["op"] == "norm":
        s["weight"], s["bias"] = affine(case["kind"], case["affine"])
        if grad:
            s["dn"] = normal(b, n, dim, leaf=False)
        return s
    s["y"] = normal(b, n, dim, std=0.7)
    s["weight"], s["bias"] = affine(case["post"], "weight" if case["post"] == "rms" else "weight_bias")
    s["next_weight"], s["next_bias"] = affine(case["next"], "weight" if case["next"] == "rms" else "weight_bias")
    shape = {"sample": (b, 1, dim), "token": (b, n, 1), "full": (b, n, dim)}.get(case["gate"])
    s["gate"] = None if shape is None else normal(*shape, mean=0.5, std=0.3)
    s["scale"] = normal(dim, dtype=param, mean=0.5, std=0.1) if case["scale"] else None
    s["key"] = key() if case["p"] else None
    if grad:
        s["dout"] = normal(b, n, dim, dtype=outer, leaf=False)
        s["dn"] = normal(b, n, dim, leaf=False) if case["next"] != "none" else None
    return s


def _inputs(s):
    names = ("x", "y", "weight", "bias", "gate", "scale", "next_weight", "next_bias")
    return {k: s[k] for k in names if s.get(k) is not None}


def _run_own(s):
    import pack3d_amd as p3d

    case = s["case"]
    if case["op"] == "norm":
        out = p3d.block_norm(s["x"], p3d.Norm(case["kind"], s["weight"], s["bias"], 1e-5),
                             dtype=TYPES[case["dtype"]][1])
        return {"n": out}, ["dn"]
    if case["op"] == "close":
        def spec(kind, weight, bias):
            return None if kind == "none" else p3d.Norm(kind, weight, bias, 1e-5)
        got = p3d.block_residual(s["x"], s["y"], post_norm=spec(case["post"], s["weight"], s["bias"]),
                                 gate=s["gate"], scale=s["scale"], alpha=case["alpha"], p=case["p"], seed=s["key"],
                                 next_norm=spec(case["next"], s["next_weight"], s["next_bias"]))
        return ({"out": got}, ["dout"]) if case["next"] == "none" else ({"out": got[0], "n": got[1]}, ["dout", "dn"])
    if case["op"] == "dropout":
        return {"y": p3d.counter_dropout(s["x"], case["p"], s["key"])}, ["dy"]
    outs = p3d.apply_rotary(s["heads"], s["positions"], s["freqs"], pairs=_axis_pairs(case), layout=case["layout"],
                            magnitude=s["magnitude"])
    return {"heads": list(outs)}, ["douts"]


# ------------------------------------------------------------- plain form

LOW = 0xFFFFFFFF


def _keep(count, p, key):
    """Truth values of what a dropout of rate p keeps of ``count`` elements: element i compares 16 of the
    generator's bits with p.  The generator is Philox4x32-10 (Salmon et al., Parallel random numbers: as easy
    as 1, 2, 3, 2011) on the counter (i // 8, offset), a block of 128 bits for eight elements."""
    group = torch.arange(-(-count // 8), device=key.device)
    c0, c1 = group & LOW, group >> 32
    c2, c3 = key[1] & LOW, (key[1] >> 32) & LOW
    k0, k1 = key[0] & LOW, (key[0] >> 32) & LOW
    for _ in range(10):
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64 bits, of which the sign is a bit like the others
        c0, c1, c2, c3 = ((m1 >> 32) & LOW) ^ c1 ^ k0, m1 & LOW, ((m0 >> 32) & LOW) ^ c3 ^ k1, m0 & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1)
    bits = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:count]
    return bits >= _threshold(p)


def _threshold(p):
    return min(65535, int(p * 65536 + 0.5))


def _dropped(x, p, key):
    kept = _keep(x.numel(), p, key).view(x.shape)
    return torch.where(kept, x * (65536 / (65536 - _threshold(p))), 0.0)


def _normed(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    x = x if weight is None else x * weight.float()
    return x if bias is None else x + bias.float()


def _turned(x, cos, sin, pairs, layout):
    if layout == "half":
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, x[..., 2 * pairs:]), -1)


def _angles(s):
    """Angles [batch or 1, 1, tokens, pairs] in 64 bits: in 32, those of far positions are off by more than the result's step."""
    case, positions = s["case"], s["positions"]
    if case["axes"] == 1:
        positions = positions[..., None]
    axis = torch.repeat_interleave(torch.arange(case["axes"]), torch.tensor(_axis_pairs(case))).to(positions.device)
    angles = positions[..., axis].double() * s["freqs"]
    return angles.view(-1, 1, *angles.shape[-2:])


def _run_plain(s):
    case = s["case"]
    outer, inner = TYPES[case["dtype"]]
    if case["op"] == "norm":
        return {"n": _normed(s["x"].float(), case["kind"], s["weight"], s["bias"]).to(inner)}, ["dn"]
    if case["op"] == "dropout":
        return {"y": _dropped(s["x"].float(), case["p"], s["key"]).to(inner)}, ["dy"]
    if case["op"] == "rotary":
        angles = _angles(s)
        cos, sin = (angles.cos() * s["magnitude"]).float(), (angles.sin() * s["magnitude"]).float()
        return {"heads": [_turned(t.float(), cos, sin, case["pairs"], case["layout"]).to(inner)
                          for t in s["heads"]]}, ["douts"]
    z = s["y"].float()
    if case["post"] != "none":
        z = _normed(z, case["post"], s["weight"], s["bias"])
    if case["p"]:
        z = _dropped(z, case["p"], s["key"])
    z = z if s["gate"] is None else z * s["gate"].float()
    z = z if s["scale"] is None else z * s["scale"].float()
    out = case["alpha"] * s["x"].float() + z
    if case["next"] == "none":
        return {"out": out.to(outer)}, ["dout"]
    n = _normed(out, case["next"], s["next_weight"], s["next_bias"])
    return {"out": out.to(outer), "n": n.to(inner)}, ["dout", "dn"]


def run(state):
    train = state["case"]["way"] == "train"
    with torch.set_grad_enabled(train):
        outs, upstream = (_run_own if own else _run_plain)(state)
    if not train:
        return outs
    if state["case"]["op"] == "rotary":
        grads = torch.autograd.grad(outs["heads"], state["heads"], state["douts"])
        return {"heads": [t.detach() for t in outs["heads"]], "grads": list(grads)}
    leaves = _inputs(state)
    grads = torch.autograd.grad(list(outs.values()), list(leaves.values()), [state[k] for k in upstream])
    return {**{k: t.detach() for k, t in outs.items()}, **{"d_" + k: g for k, g in zip(leaves, grads)}}


def work(case):
    outer, inner = (torch.finfo(t).bits // 8 for t in TYPES[case["dtype"]])
    b, n, train = case["batch"], case["tokens"], case["way"] == "train"
    if case["op"] == "rotary":
        count = b * n * case["head_dim"] * (case["heads"] + case["keys"] * case["kv_heads"])
        turned = count // case["head_dim"] * case["pairs"]
        return {"bytes": count * inner * 2 * (1 + train) + 8 * n * (3 if case["axes"] == 3 else b),
                "flops": turned * 6 * (1 + train)}
    count, dim = b * n * case["dim"], case["dim"]
    if case["op"] == "dropout":
        return {"bytes": count * inner * 2 * (1 + train) + 16, "flops": count * 2 * (1 + train)}
    param = 4 if outer == 4 else inner
    if case["op"] == "norm":
        params = param * dim * {"weight_bias": 2, "weight": 1, "none": 0}[case["affine"]]
        return {"bytes": count * (outer + inner) * (1 + train) + params * (1 + train),
                "flops": count * (8 + 14 * train)}
    after = case["next"] != "none"
    gates = {"none": 0, "sample": b * dim, "token": b * n, "full": count}[case["gate"]] * inner
    params = param * dim * (2 * (case["post"] == "layer") + (case["post"] == "rms") + 2 * (case["next"] == "layer")
                            + (case["next"] == "rms") + case["scale"])
    once = count * (2 * outer + inner + after * inner) + gates + params  # x, y, gate and parameters in, out and n out
    again = count * (2 * outer + inner + after * inner) + gates + params  # dout and dn in, dx, dy and the others out
    return {"bytes": once + train * again, "flops": count * (16 + 12 * after + train * (24 + 14 * after))}


# ----------------------------------------------------- definition in 64 bits

def _philox_words(groups, key):
    """The generator's four words for each counter of the array, in unsigned 64-bit arithmetic."""
    low, shift = np.uint64(LOW), np.uint64(32)
    seed, offset = (np.uint64(int(v) & (2 ** 64 - 1)) for v in key)
    c = [groups & low, groups >> shift, np.full_like(groups, offset & low), np.full_like(groups, offset >> shift)]
    k = [int(seed & low), int(seed >> shift)]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> shift) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> shift) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def _factor64(shape, p, key):
    """What dropout multiplies each element by: 0, or the reciprocal of the rate that stays."""
    count, step, parts = math.prod(shape), 1 << 17, []
    key = key.tolist()
    for at in range(0, -(-count // 8), step):
        words = _philox_words(np.arange(at, min(at + step, -(-count // 8)), dtype=np.uint64), key)
        words = np.stack([w.astype(np.uint32) for w in words], -1)
        parts.append(words.view(np.uint16).reshape(-1) >= _threshold(p))  # the low half first
    kept = torch.from_numpy(np.concatenate(parts)[:count]).to(DEVICE)
    return kept.double().view(shape) / (1.0 - _threshold(p) / 65536)


def _stats64(x, kind):
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    rstd = ((x - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    return (x - mean) * rstd, rstd


def _norm_back64(d, hat, rstd, kind, weight):
    """(dx, dweight, dbias) for the gradient d of hat * weight + bias."""
    g = d if weight is None else d * weight.double()
    dx = g - hat * (g * hat).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - g.mean(-1, keepdim=True)
    return dx * rstd, (d * hat).sum((0, 1)), d.sum((0, 1))


def _affine64(hat, weight, bias):
    hat = hat if weight is None else hat * weight.double()
    return hat if bias is None else hat + bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    train = case["way"] == "train"
    with torch.no_grad():
        return _exact(case, s, train)


def _exact(case, s, train):
    if case["op"] == "rotary":
        p, half = case["pairs"], case["layout"] == "half"
        first = torch.arange(p, device=DEVICE) if half else 2 * torch.arange(p, device=DEVICE)
        second = first + (p if half else 1)
        turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEVICE), _angles(s))

        def turned(x, turn):
            out = x.double()
            z = torch.complex(out[..., first], out[..., second]) * turn
            out[..., first], out[..., second] = z.real, z.imag
            return out
        outs = {"heads": [turned(t, turn) for t in s["heads"]]}
        return {**outs, "grads": [turned(t, turn.conj()) for t in s["douts"]]} if train else outs
    if case["op"] == "dropout":
        factor = _factor64(s["x"].shape, case["p"], s["key"])
        return {"y": s["x"].double() * factor, **({"d_x": s["dy"].double() * factor} if train else {})}
    x = s["x"].double()
    if case["op"] == "norm":
        hat, rstd = _stats64(x, case["kind"])
        outs = {"n": _affine64(hat, s["weight"], s["bias"])}
        if train:
            grads = _norm_back64(s["dn"].double(), hat, rstd, case["kind"], s["weight"])
            outs.update({"d_" + k: g for k, g in zip(("x", "weight", "bias"), grads) if s[k] is not None})
        return outs
    y = s["y"].double()
    hat, rstd = (y, None) if case["post"] == "none" else _stats64(y, case["post"])
    z = _affine64(hat, s["weight"], s["bias"])
    factor = _factor64(y.shape, case["p"], s["key"]) if case["p"] else torch.ones((), dtype=torch.float64, device=DEVICE)
    z = z * factor
    gate = torch.ones((), dtype=torch.float64, device=DEVICE) if s["gate"] is None else s["gate"].double()
    scale = torch.ones((), dtype=torch.float64, device=DEVICE) if s["scale"] is None else s["scale"].double()
    out = case["alpha"] * x + gate * scale * z
    outs, back = {"out": out}, {}
    if case["next"] != "none":
        after, after_rstd = _stats64(out, case["next"])
        outs["n"] = _affine64(after, s["next_weight"], s["next_bias"])
    if not train:
        return outs
    d = s["dout"].double()
    if case["next"] != "none":
        dx, back["next_weight"], back["next_bias"] = _norm_back64(s["dn"].double(), after, after_rstd, case["next"],
                                                                 s["next_weight"])
        d = d + dx
    back["x"] = case["alpha"] * d
    back["scale"] = (d * gate * z).sum((0, 1))
    if s["gate"] is not None:
        back["gate"] = d * scale * z
        for i in (1, 2):
            if s["gate"].shape[i] == 1:
                back["gate"] = back["gate"].sum(i, keepdim=True)
    d = d * gate * scale * factor
    back["y"] = d
    if case["post"] != "none":
        back["y"], back["weight"], back["bias"] = _norm_back64(d, hat, rstd, case["post"], s["weight"])
    return {**outs, **{"d_" + k: back[k] for k in _inputs(s)}}
