"""What surrounds an attention or feed-forward block: the norm before it, and its end
in one pass.

``block_norm`` is a LayerNorm or RMSNorm of any width up to 8,192.
``block_residual`` is everything between a block's last product and the next block:

    out = alpha * x + scale * gate * dropout(post_norm(y)),    n = next_norm(out)

x the residual stream, y the block's output; post_norm, dropout, gate, scale and
next_norm each optional.  In torch operations that is a pass over the tokens for
each step, forward and backward; here x and y are read once and out and n written
once (``p3d_block_fwd``), and the backward reads the gradients, x and y once
(``p3d_block_bwd``).  Sums and statistics are fp32, each output is rounded once,
parameter gradients are summed in a fixed order.

``PACK3DAttention`` takes the same choices for its own end (post_norm, layer_scale,
dropout) and, per call, gate, next_norm and an input that is already normalised.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .dropout import mask_args

MAX_DIM = 8192
MAX_STRIDE = 2 ** 29  # elements between rows
KINDS = {"layer": 1, "rms": 2}  # enum p3d_norm_kind
SAMPLE, TOKEN, FULL = 1, 2, 3   # enum p3d_gate_kind


class Norm(NamedTuple):
    """LayerNorm ("layer") or RMSNorm ("rms") with weight and bias [dim] or None."""

    kind: str = "layer"
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-5

    @classmethod
    def of(cls, module):
        """The norm of a torch.nn.LayerNorm or RMSNorm over the last dimension."""
        if not isinstance(module, (torch.nn.LayerNorm, torch.nn.RMSNorm)) or len(module.normalized_shape) != 1:
            raise ValueError("Norm.of takes an nn.LayerNorm or nn.RMSNorm over the last dimension")
        if isinstance(module, torch.nn.LayerNorm):
            return cls("layer", module.weight, module.bias, module.eps)
        # nn.RMSNorm without eps takes that of the type it computes in, fp32 here.
        return cls("rms", module.weight, None, torch.finfo(torch.float32).eps if module.eps is None else module.eps)


def _rows(t, dim):
    """t as rows [*, dim] with unit channel stride (a copy where it does not lie so), and the row stride."""
    t = t.reshape(-1, dim)
    if (dim > 1 and t.stride(1) != 1) or t.stride(0) >= MAX_STRIDE:
        t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(0)


def _split(samples, tokens, dim, backward):
    """(ranges that a sample's rows are cut into, workgroups)."""
    threads = next((t for t, most in ((8, 64), (16, 128), (32, 256), (64, 512), (128, 1024), (256, 2048))
                    if dim <= most), 512)  # of a row
    rows = max(1, 256 // threads) if threads <= 64 else 1  # that a workgroup holds at a time
    steps = -(-tokens // rows) * samples
    if backward:
        # One round of what the GPU runs at a time (two waves a SIMD): each workgroup
        # leaves a row of partial parameter gradients.
        wanted = (1 << 17) // (threads if threads > 64 else 256)
    elif threads > 64:
        wanted = (1 << 18) // threads
    else:
        # Several rounds, of at least four steps each once every CU has work: a workgroup
        # begins by loading the parameters (4,913 x 3 rows of 327: 21 us in 921, 25 in 3,685).
        wanted = max(min(1024, steps), min(4096, steps // 4))
    splits = max(1, min(wanted // samples, -(-tokens // rows)))
    return splits, min(splits * samples, wanted)


def _check_norm(name, norm, dim, device):
    if norm is None:
        return
    if not isinstance(norm, Norm) or norm.kind not in KINDS:
        raise ValueError(f"{name} must be a Norm of kind layer or rms")
    if not (math.isfinite(norm.eps) and norm.eps >= 0):
        raise ValueError(f"{name}: eps must be finite and not negative")
    for t in (norm.weight, norm.bias):
        _check_param(name, t, dim, device)


def _check_param(name, t, dim, device):
    if t is not None and (t.shape != (dim,) or t.device != device or not t.is_floating_point()):
        raise ValueError(f"{name}: parameters must be floating point [dim] on the input's device")


def _gate_kind(gate, x):
    """How the gate spreads over x [batch, tokens, dim] or [tokens, dim]."""
    if gate is None:
        return 0
    if gate.ndim != x.ndim or gate.device != x.device or gate.dtype not in _lib.DTYPES:
        raise ValueError("gate must be fp32, fp16 or bf16 with x's number of dimensions, on its device")
    *lead, n, dim = x.shape
    if gate.shape == (*lead, n, dim):
        return FULL
    if gate.shape == (*lead, n, 1):
        return TOKEN
    if gate.shape == (*lead, 1, dim) or gate.shape == (*(1 for _ in lead), 1, dim):
        return SAMPLE
    raise ValueError("gate must be [batch or 1, 1, dim], [batch, tokens, 1] or [batch, tokens, dim]")


class _Call:
    """One forward: the argument block of both directions and what it points into."""

    def __init__(self, x, y, gate, scale, params, kinds, eps, alpha, mask, gate_kind, inner):
        dim = x.shape[-1]
        a = _lib.BlockArgs()
        self.shape, self.dim, self.args = x.shape, dim, a
        rows = x.numel() // dim if dim else 0
        self.rows = rows
        # Rows that share a gate vector; a gate of batch 1 is shared by all of them.
        a.samples = gate.shape[0] if gate_kind == SAMPLE and x.ndim == 3 else 1
        a.tokens = rows // a.samples if rows else 0
        a.dim = dim
        a.outer, a.inner = _lib.DTYPES[x.dtype], _lib.DTYPES[inner]
        given = [t for t in (*params, scale) if t is not None]
        dtype = given[0].dtype if given and all(t.dtype == given[0].dtype for t in given) else torch.float32
        dtype = dtype if dtype in _lib.DTYPES else torch.float32
        a.param = _lib.DTYPES[dtype]
        self.keep = [None if t is None else t.to(dtype).contiguous() for t in (*params, scale)]
        w1, b1, w2, b2, sc = (_lib.ptr(t) for t in self.keep)
        a.post, a.next = _lib.NormArgs(w1, b1, kinds[0], eps[0]), _lib.NormArgs(w2, b2, kinds[1], eps[1])
        a.scale, a.alpha, a.dropout = sc, alpha, mask
        self.bind(x, y, gate)
        a.gate_kind = gate_kind
        self.inner = inner

    def bind(self, x, y, gate):
        """Points the arguments at x, y and the gate."""
        a, dim = self.args, self.dim
        x, a.x_stride = _rows(x, dim)
        a.x = x.data_ptr()
        self.tensors = [x]
        if y is not None:
            y, a.y_stride = _rows(y, dim)
            a.y = y.data_ptr()
            self.tensors.append(y)
        if gate is not None:
            gate, a.gate_stride = _rows(gate, gate.shape[-1])
            a.gate, a.gate_dtype = gate.data_ptr(), _lib.DTYPES[gate.dtype]
            self.tensors.append(gate)

    def forward(self, x, has_y, save):
        a, dev = self.args, x.device
        out = torch.empty(self.shape, dtype=x.dtype, device=dev) if has_y else None
        n = torch.empty(self.shape, dtype=self.inner, device=dev) if a.next.kind else None
        stats = torch.empty(4, self.rows, dtype=torch.float32, device=dev) if save else None
        if self.rows:
            a.out, a.n, a.stats = _lib.ptr(out), _lib.ptr(n), _lib.ptr(stats)
            a.splits, a.grid = _split(a.samples, a.tokens, self.dim, False)
            _lib.launch("p3d_block_fwd", dev, a)
        return out, n, stats


class _Block(torch.autograd.Function):
    """block_norm and block_residual under autograd.  The forward saves its inputs and
    the rows' statistics; the backward forms out again from x and y."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, w1, b1, w2, b2, state, made):
        call = _Call(x, y, gate, scale, (w1, b1, w2, b2), *made)
        out, n, stats = call.forward(x, y is not None, True)
        ctx.save_for_backward(x, y, gate, scale, w1, b1, w2, b2, state, stats)
        ctx.made = made
        ctx.set_materialize_grads(False)
        return (out, n) if out is not None and n is not None else (n if out is None else out)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, y, gate, scale, w1, b1, w2, b2, state, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        has_next = bool(ctx.made[0][1])
        dout, dn = grads if len(grads) == 2 else ((None, grads[0]) if y is None else (grads[0], None))
        none = (None,) * 10
        if dout is None and dn is None:
            return none
        params = (w1, b1, scale, w2, b2)
        wanted = [t is not None and need[i] for t, i in zip(params, (4, 5, 3, 6, 7))]
        alpha, gate_kind = ctx.made[2], ctx.made[4]
        call = _Call(x, y, gate, scale, (w1, b1, w2, b2), *ctx.made)
        a, dim, dev, f32 = call.args, call.dim, x.device, torch.float32
        # Without a gradient through the next norm dx is alpha dout: dout itself for 1.
        through = dn is None and alpha == 1.0
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] and not through else None
        dy = torch.empty(y.shape, dtype=y.dtype, device=dev) if y is not None and need[1] else None
        dgate = part = dgate_part = None
        if gate is not None and need[2] and gate_kind != SAMPLE:
            dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
        sums = []
        if call.rows:
            a.splits, a.grid = _split(a.samples, a.tokens, dim, True)
            if gate is not None and need[2] and gate_kind == SAMPLE:
                dgate_part = torch.empty(a.splits, a.samples * dim, dtype=f32, device=dev)
                dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
                sums.append((dgate_part, dgate))
            if any(wanted):
                part = torch.empty(a.grid, 5, dim, dtype=f32, device=dev)
            keep = []
            for name, t, dtype in (("dout", dout, x.dtype), ("dn", dn, call.inner)):
                if t is not None:
                    t, stride = _rows(t.to(dtype), dim)
                    keep.append(t)
                    setattr(a, name, t.data_ptr())
                    setattr(a, name + "_stride", stride)
            a.stats, a.dx, a.dy, a.part = stats.data_ptr(), _lib.ptr(dx), _lib.ptr(dy), _lib.ptr(part)
            a.dgate_part = _lib.ptr(dgate_part)
            a.dgate = _lib.ptr(dgate) if gate_kind in (TOKEN, FULL) else None
            if dx is not None or dy is not None or dgate is not None or part is not None:
                _lib.launch("p3d_block_bwd", dev, a)
        elif gate is not None and need[2]:
            dgate = torch.zeros_like(gate)
        out = [None] * 5
        for i, (t, want) in enumerate(zip(params, wanted)):
            if not want:
                continue
            if not call.rows or (i >= 3 and dn is None):
                out[i] = torch.zeros_like(t)
                continue
            out[i] = torch.empty(dim, dtype=t.dtype if t.dtype in _lib.DTYPES else f32, device=dev)
            sums.append((part[:, i], out[i]))
        if sums:
            with torch.cuda.device(dev):
                _lib.sum_rows(sums, dev)
        dw1, db1, dscale, dw2, db2 = (g if g is None else g.to(t.dtype) for g, t in zip(out, params))
        if through and need[0]:
            dx = dout
        return dx, dy, dgate, dscale, dw1, db1, dw2, db2, None, None


def _run(x, y, gate, scale, post, after, alpha, p, seed, inner):
    mask, state = mask_args(p, seed, x.device)
    gate_kind = _gate_kind(gate, x)
    norms = [n if n is not None else Norm() for n in (post, after)]
    kinds = [0 if n is None else KINDS[n.kind] for n in (post, after)]
    params = [t for n in norms for t in (n.weight, n.bias)]
    made = (kinds, [n.eps for n in norms], alpha, mask, gate_kind, inner)
    inputs = (x, y, gate, scale, *params)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        return _Block.apply(*inputs, state, made)
    out, n, _ = _Call(x, y, gate, scale, params, *made).forward(x, y is not None, False)
    return (out, n) if out is not None and n is not None else (n if out is None else out)


def _check_x(x):
    _lib.require_device(x, "x")
    if x.dtype not in _lib.DTYPES:
        raise ValueError("x must be fp32, fp16 or bf16")
    if x.ndim not in (2, 3) or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError("x must be [batch, tokens, dim] or [tokens, dim] with dim 1 to 8192")
    if x.numel() // x.shape[-1] >= 2 ** 31:
        raise ValueError("x has too many rows")


def block_norm(x, norm: Norm, *, dtype=None):
    """``norm`` of x [batch, tokens, dim] or [tokens, dim] in ``dtype`` (x's own; for an
    fp32 x also fp16 or bf16, as the next products take it): statistics in fp32, one
    rounding, any row stride.  Differentiable in x and the norm's parameters."""
    _check_x(x)
    if norm is None:
        raise ValueError("block_norm needs a Norm")
    _check_norm("norm", norm, x.shape[-1], x.device)
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _lib.DTYPES or (x.dtype != torch.float32 and dtype != x.dtype):
        raise ValueError("dtype must be x's, or fp16 or bf16 for an fp32 x")
    return _run(x, None, None, None, None, norm, 1.0, 0.0, None, dtype)


def block_residual(x, y, *, post_norm: Optional[Norm] = None, gate=None, scale=None, alpha=1.0, p=0.0, seed=None,
                   next_norm: Optional[Norm] = None):
    """The end of a block: ``alpha * x + scale * gate * dropout(post_norm(y))``, and with
    ``next_norm`` the pair of that sum and its norm, from one pass over the rows.

    x, y: [batch, tokens, dim] or [tokens, dim]; y has x's type or, over an fp32 x, fp16
    or bf16.  The sum has x's type, the norm y's (computed from the unrounded sum).
    gate: [batch or 1, 1, dim] (per sample), [batch, tokens, 1] or [batch, tokens, dim].
    scale: [dim], per channel.  p, seed: as counter_dropout's, on y's elements.
    Differentiable in x, y, gate, scale and the norms' parameters (first order)."""
    _check_x(x)
    if y.shape != x.shape or y.device != x.device:
        raise ValueError("y must have x's shape and device")
    if y.dtype not in _lib.DTYPES or (x.dtype != torch.float32 and y.dtype != x.dtype):
        raise ValueError("y must have x's type, or fp16 or bf16 over an fp32 x")
    dim = x.shape[-1]
    _check_norm("post_norm", post_norm, dim, x.device)
    _check_norm("next_norm", next_norm, dim, x.device)
    _check_param("scale", scale, dim, x.device)
    alpha = float(alpha)
    if not math.isfinite(alpha):
        raise ValueError("alpha must be finite")
    return _run(x, y, gate, scale, post_norm, next_norm, alpha, p, seed, y.dtype)
