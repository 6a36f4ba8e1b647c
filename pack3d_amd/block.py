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
_NO_MASK = _lib.Dropout(None, 0, 0, 0, 0)


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
    if t.is_contiguous():
        return t, dim
    t = t.reshape(-1, dim)
    if (dim > 1 and t.stride(1) != 1) or t.stride(0) >= MAX_STRIDE:
        t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(0)


def _split(samples, tokens, dim, backward):
    """(ranges that a sample's rows are cut into, workgroups)."""
    threads = 8  # of a row
    while threads < 512 and dim > threads * 8:
        threads *= 2
    rows = 256 // threads if threads <= 64 else 1  # that a workgroup holds at a time
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
    if not isinstance(norm, Norm) or norm.kind not in KINDS:
        raise ValueError(f"{name} must be a Norm of kind layer or rms")
    if not 0 <= norm.eps < math.inf:
        raise ValueError(f"{name}: eps must be finite and not negative")
    if norm.weight is not None:
        _check_param(name, norm.weight, dim, device)
    if norm.bias is not None:
        _check_param(name, norm.bias, dim, device)


def _check_param(name, t, dim, device):
    if t.shape != (dim,) or t.device != device or not t.is_floating_point():
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


class _Spec(NamedTuple):
    """What a call computes, apart from its tensors."""

    kinds: tuple      # of the post and the next norm, 0 where there is none
    eps: tuple
    alpha: float
    mask: object      # ctypes block of the dropout mask
    gate_kind: int
    inner: torch.dtype


def _bind(spec, x, y, gate, scale, params):
    """The argument block of both directions, without outputs; and what it points into
    besides the tensors given (copies of those that do not lie as the kernels read them)."""
    a, keep = _lib.BlockArgs(), []
    dim = x.shape[-1]
    rows = x.numel() // dim
    dtypes = _lib.DTYPES
    a.dim, a.alpha, a.dropout = dim, spec.alpha, spec.mask
    a.outer, a.inner = dtypes[x.dtype], dtypes[spec.inner]
    t, a.x_stride = _rows(x, dim)
    a.x = t.data_ptr()
    keep.append(t)
    if y is not None:
        t, a.y_stride = _rows(y, dim)
        a.y = t.data_ptr()
        keep.append(t)
    samples = 1  # runs of rows that share a gate vector; a gate of batch 1 is shared by all of them
    if gate is not None:
        if spec.gate_kind == SAMPLE and x.ndim == 3:
            samples = gate.shape[0]
        t, a.gate_stride = _rows(gate, gate.shape[-1])
        a.gate, a.gate_dtype, a.gate_kind = t.data_ptr(), dtypes[gate.dtype], spec.gate_kind
        keep.append(t)
    a.samples, a.tokens = samples, rows // samples
    given = [t for t in (*params, scale) if t is not None]
    if given:
        # One type for all: their own, or fp32, which holds each of them exactly.
        dtype = given[0].dtype
        if dtype not in dtypes or any(t.dtype != dtype for t in given):
            dtype = torch.float32
        a.param = dtypes[dtype]
        at = []
        for t in (*params, scale):
            if t is not None and (t.dtype != dtype or not t.is_contiguous()):
                t = t.to(dtype).contiguous()
                keep.append(t)
            at.append(None if t is None else t.data_ptr())
        w1, b1, w2, b2, a.scale = at
    else:
        w1 = b1 = w2 = b2 = None
    kinds, eps = spec.kinds, spec.eps
    if kinds[0]:
        a.post = _lib.NormArgs(w1, b1, kinds[0], eps[0])
    if kinds[1]:
        a.next = _lib.NormArgs(w2, b2, kinds[1], eps[1])
    return a, keep


def _empty(like, dtype):
    """A contiguous tensor of like's shape."""
    if like.is_contiguous():
        return torch.empty_like(like, dtype=dtype)
    return torch.empty(like.shape, dtype=dtype, device=like.device)


def _forward(spec, x, y, gate, scale, params, save):
    """(out or None, n or None, the argument block with what it points into, statistics or None)."""
    a, keep = _bind(spec, x, y, gate, scale, params)
    rows = a.samples * a.tokens
    out = None if y is None else _empty(x, x.dtype)
    n = _empty(x, spec.inner) if spec.kinds[1] else None
    stats = torch.empty(4, rows, dtype=torch.float32, device=x.device) if save else None
    if rows:
        if out is not None:
            a.out = out.data_ptr()
        if n is not None:
            a.n = n.data_ptr()
        if save:
            a.stats = stats.data_ptr()
        a.splits, a.grid = _split(a.samples, a.tokens, a.dim, False)
        _lib.launch("p3d_block_fwd", x.device, a)
    return out, n, (a, keep), stats


def _still(a, x, y, gate, scale, params):
    """Whether an argument block points at these very tensors (saved tensors may come back as others)."""
    if a.x != x.data_ptr() or a.y != (None if y is None else y.data_ptr()):
        return False
    post, after = a.post, a.next
    for at, t in ((a.gate, gate), (a.scale, scale), (post.weight, params[0]), (post.bias, params[1]),
                  (after.weight, params[2]), (after.bias, params[3])):
        if at != (None if t is None else t.data_ptr()):
            return False
    return True


def _param_grads(a, params, wanted, dim):
    """Gradients of the parameters that are wanted, in the order of the argument block, and
    their addresses entered there: one allocation where they have one type."""
    which = [i for i in range(5) if wanted[i]]
    grads = [None] * 5
    if not which:
        return grads
    dtype = params[which[0]].dtype
    if dtype in _lib.DTYPES and all(params[i].dtype == dtype for i in which):
        made = torch.empty(len(which) * dim, dtype=dtype, device=params[which[0]].device).split(dim)
    else:
        made = [torch.empty_like(params[i], dtype=params[i].dtype if params[i].dtype in _lib.DTYPES else torch.float32,
                                 memory_format=torch.contiguous_format) for i in which]
    to, types = a.d_param, a.d_param_dtype
    for i, g in zip(which, made):
        grads[i], to[i], types[i] = g, g.data_ptr(), _lib.DTYPES[g.dtype]
    return grads


class _Block(torch.autograd.Function):
    """block_norm and block_residual under autograd.  The forward saves its inputs and
    the rows' statistics; the backward forms out again from x and y."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, w1, b1, w2, b2, state, spec):
        out, n, ctx.call, ctx.stats = _forward(spec, x, y, gate, scale, (w1, b1, w2, b2), True)
        ctx.save_for_backward(x, y, gate, scale, w1, b1, w2, b2, state)
        ctx.spec = spec
        ctx.set_materialize_grads(False)
        return (out, n) if out is not None and n is not None else (n if out is None else out)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, y, gate, scale, w1, b1, w2, b2, _ = ctx.saved_tensors
        need, spec, (a, keep) = ctx.needs_input_grad, ctx.spec, ctx.call
        dout, dn = grads if len(grads) == 2 else ((None, grads[0]) if y is None else (grads[0], None))
        if dout is None and dn is None:
            return (None,) * 10
        if _still(a, x, y, gate, scale, (w1, b1, w2, b2)):
            a = _lib.BlockArgs.from_buffer_copy(a)
        else:
            a, keep = _bind(spec, x, y, gate, scale, (w1, b1, w2, b2))
        dim, rows = a.dim, a.samples * a.tokens
        # Without a gradient through the next norm dx is alpha dout: dout itself for 1.
        through = dn is None and spec.alpha == 1.0
        dx = dy = dgate = None
        if not through and (need[0] or dn is not None):
            dx = _empty(x, x.dtype)
            a.dx = dx.data_ptr()
        if y is not None:
            dy = _empty(y, y.dtype)
            a.dy = dy.data_ptr()
        if gate is not None and (need[2] or spec.gate_kind != SAMPLE):
            dgate = _empty(gate, gate.dtype)
            a.dgate = dgate.data_ptr()
        params = (w1, b1, scale, w2, b2)
        wanted = (need[4] and w1 is not None, need[5] and b1 is not None, need[3] and scale is not None,
                  need[6] and w2 is not None, need[7] and b2 is not None)
        if rows:
            after = dn is not None
            dparams = _param_grads(a, params, wanted if after else (*wanted[:3], False, False), dim)
            if not after and (wanted[3] or wanted[4]):
                dparams = [torch.zeros_like(t) if w and g is None else g for g, t, w in zip(dparams, params, wanted)]
            a.splits, a.grid = _split(a.samples, a.tokens, dim, True)
            work = torch.empty((a.grid * 5 + (a.splits * a.samples if spec.gate_kind == SAMPLE else 0)) * dim,
                               dtype=torch.float32, device=x.device)
            if y is not None:
                if dout is None:  # only n was used: a row of zeros, for every row
                    dout = torch.zeros(1, dim, dtype=x.dtype, device=x.device).expand(rows, dim)
                dout, a.dout_stride = _rows(dout if dout.dtype == x.dtype else dout.to(x.dtype), dim)
                a.dout = dout.data_ptr()
            if after:
                dn, a.dn_stride = _rows(dn if dn.dtype == spec.inner else dn.to(spec.inner), dim)
                a.dn = dn.data_ptr()
            a.stats, a.work = ctx.stats.data_ptr(), work.data_ptr()
            _lib.launch("p3d_block_bwd", x.device, a)
        else:
            dparams = [torch.zeros_like(t) if w else None for t, w in zip(params, wanted)]
            if dgate is not None:
                dgate.zero_()
        dw1, db1, dscale, dw2, db2 = (g if g is None or g.dtype == t.dtype else g.to(t.dtype)
                                      for g, t in zip(dparams, params))
        return ((grads[0] if through else dx) if need[0] else None, dy if need[1] else None,
                dgate if need[2] else None, dscale, dw1, db1, dw2, db2, None, None)


def _run(x, y, gate, scale, post, after, alpha, p, seed, inner):
    mask, state = mask_args(p, seed, x.device) if p != 0.0 else (_NO_MASK, None)
    gate_kind = _gate_kind(gate, x)
    w1, b1, w2, b2 = params = ((None, None) if post is None else post[1:3]) + ((None, None) if after is None else after[1:3])
    spec = _Spec((0 if post is None else KINDS[post.kind], 0 if after is None else KINDS[after.kind]),
                 (0.0 if post is None else post.eps, 0.0 if after is None else after.eps), alpha, mask, gate_kind, inner)
    if torch.is_grad_enabled():
        for t in (x, y, gate, scale, *params):
            if t is not None and t.requires_grad:
                return _Block.apply(x, y, gate, scale, w1, b1, w2, b2, state, spec)
    out, n, _, _ = _forward(spec, x, y, gate, scale, params, False)
    return n if out is None else out if n is None else (out, n)


def _check_x(x):
    if not x.is_cuda:
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
    if post_norm is not None:
        _check_norm("post_norm", post_norm, dim, x.device)
    if next_norm is not None:
        _check_norm("next_norm", next_norm, dim, x.device)
    if scale is not None:
        _check_param("scale", scale, dim, x.device)
    alpha = float(alpha)
    if not math.isfinite(alpha):
        raise ValueError("alpha must be finite")
    return _run(x, y, gate, scale, post_norm, next_norm, alpha, p, seed, y.dtype)
