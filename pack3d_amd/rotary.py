"""Rotary positions of queries and keys: interleaved or half layout, whole heads or
part of them, one to three axes of coordinates, frequencies scaled for grids and
sequences beyond those of training.

``apply_rotary`` turns up to four tensors in one launch (``p3d_rotary``): before
``pack3d_hip``, which takes rotated q, kl and kg, or anywhere else.  The layer's
own rotation (``rope.py``) is fused into its kernels, for whole interleaved heads
and frequencies as trained.  ``rotary_frequencies`` makes the frequencies;
``RotaryEncoding`` holds a choice of all this for ``PACK3DAttention``.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rope import _cached

LAYOUTS = ("interleaved", "half")
SCALINGS = ("none", "linear", "ntk", "parts")
MAX_TENSORS = 4


def rotary_frequencies(pairs, *, base=10000.0, scaling="none", factor=1.0, trained=None, fast=32.0, slow=1.0):
    """(frequencies, magnitude): radians a position of each pair, float64 [sum(pairs)]
    on the CPU, for the pair counts of one to three axes (an int: one axis).

    Pair j of an axis of c pairs turns by base^(-j / c).  For positions up to
    ``factor`` times those of training: "linear" divides every frequency by factor
    (positions interpolated); "ntk" raises the base to base * factor^(c / (c - 1)),
    which interpolates the slowest pair by factor and leaves the fastest; "parts"
    interpolates a pair by how often it turns over the ``trained`` positions: whole
    below ``slow`` turns, not at all above ``fast``, in between in proportion, and
    gives the magnitude 0.1 ln(factor) + 1 (Peng et al., YaRN, 2023)."""
    pairs = (pairs,) if type(pairs) is int else tuple(pairs)
    if not 1 <= len(pairs) <= 3 or any(type(c) is not int or c < 0 for c in pairs) or sum(pairs) < 1:
        raise ValueError("pairs must be one to three counts of rotary pairs")
    if scaling not in SCALINGS:
        raise ValueError("scaling must be none, linear, ntk or parts")
    if not (math.isfinite(base) and base > 1 and math.isfinite(factor) and factor >= 1):
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling == "parts" and not (trained is not None and trained > 0 and fast > slow > 0):
        raise ValueError("scaling by parts needs the trained length, and fast > slow > 0")
    made, magnitude = [], 1.0
    for count in pairs:
        j = torch.arange(count, dtype=torch.float64)
        b = base * factor ** (count / max(1, count - 1)) if scaling == "ntk" else base
        freq = b ** (-j / max(1, count))
        if scaling == "linear":
            freq = freq / factor
        elif scaling == "parts":
            kept = ((trained * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
            freq = freq * kept + freq / factor * (1.0 - kept)
            magnitude = 0.1 * math.log(factor) + 1.0
        made.append(freq)
    return torch.cat(made), magnitude


def _plan(tensors, positions, freqs, pairs, layout, magnitude):
    """Checks of apply_rotary's arguments; the argument block without the tensors, and
    the frequencies as it points at them."""
    if not 1 <= len(tensors) <= MAX_TENSORS:
        raise ValueError("apply_rotary takes one to four tensors")
    first = tensors[0]
    shape, dtype, device = first.shape, first.dtype, first.device
    if len(shape) != 4:
        raise ValueError("tensors must be [batch, heads, tokens, head_dim]")
    b, _, n, d = shape
    for t in tensors:
        if t.dtype != dtype or t.device != device or t.shape != (b, t.shape[1], n, d):
            raise ValueError("tensors must be [batch, heads, tokens, head_dim] of one type, alike but for the heads")
        if not 0 < t.shape[1] * (d // 8 + 2) <= 8192:
            raise ValueError("heads must be at least 1, heads * (head_dim / 8 + 2) at most 8192")
    if not first.is_cuda:
        _lib.require_device(first, "q and k")
    if dtype not in _lib.DTYPES:
        raise ValueError("apply_rotary takes fp32, fp16 or bf16")
    if freqs.dtype != torch.float64 or freqs.ndim != 1 or freqs.device != device:
        raise ValueError("freqs must be float64 [pairs] on the tensors' device (rotary_frequencies)")
    count = freqs.shape[0]
    if not 1 <= count <= d // 2 or d > 1024:
        raise ValueError("freqs must have 1 to head_dim / 2 pairs, head_dim at most 1024")
    a = _lib.RotaryArgs()
    axes = 1
    if pairs is None:
        a.axis_pairs[0] = count
    else:
        axes = len(pairs)
        if not 1 <= axes <= 3 or sum(pairs) != count:
            raise ValueError("pairs must give each of one to three axes its count of freqs")
        for i, c in enumerate(pairs):
            if type(c) is not int or c < 0:
                raise ValueError("pairs must be counts")
            a.axis_pairs[i] = c
    if layout not in LAYOUTS:
        raise ValueError("layout must be interleaved or half")
    if not math.isfinite(magnitude):
        raise ValueError("magnitude must be finite")
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != device:
        raise ValueError("positions must be int32 or int64 on the tensors' device")
    of, strides = positions.shape, positions.stride()
    if axes == 1:
        of, strides = (*of, 1), (*strides, 1)
    if len(of) == 2:
        of, strides = (1, *of), (0, *strides)
    if len(of) != 3 or of[0] not in (1, b) or of[1:] != (n, axes):
        raise ValueError("positions must be [tokens] or [batch, tokens], with an axis dimension last for several axes")
    a.tokens, a.count, a.batch, a.head_dim, a.pairs, a.axes = n, len(tensors), b, d, count, axes
    a.positions = positions.data_ptr()
    a.pos_sb, a.pos_sn, a.pos_sa = 0 if of[0] == 1 else strides[0], strides[1], strides[2]
    freqs = freqs.contiguous()
    a.freqs = freqs.data_ptr()
    a.pos_is64, a.half, a.dtype = positions.dtype == torch.int64, layout == "half", _lib.DTYPES[dtype]
    a.magnitude = magnitude
    return a, freqs


def _turn(plan, tensors, inverse):
    """The tensors turned, dense, with their dimensions in memory in the order of the inputs'."""
    outs, keep = [], []
    plan.inverse = inverse
    for i, t in enumerate(tensors):
        s = t.stride()
        if s[3] != 1:
            t = t.contiguous()
            keep.append(t)
            s = t.stride()
        out = torch.empty_like(t)
        o = out.stride()
        if o[3] != 1:
            out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
            o = out.stride()
        plan.x[i] = _lib.View(t.data_ptr(), s[0], s[1], s[2])
        plan.y[i] = _lib.View(out.data_ptr(), o[0], o[1], o[2])
        plan.heads[i] = t.shape[1]
        outs.append(out)
    if tensors[0].numel():
        _lib.launch("p3d_rotary", tensors[0].device, plan)
    return tuple(outs)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, positions, freqs, *tensors):
        ctx.plan = plan
        ctx.save_for_backward(positions, freqs)
        return _turn(plan, tensors, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        ctx.saved_tensors  # raises where positions or freqs were changed since the forward
        need = [i for i in range(len(grads)) if ctx.needs_input_grad[3 + i]]
        plan = _lib.RotaryArgs.from_buffer_copy(ctx.plan)
        plan.count = len(need)
        back = dict(zip(need, _turn(plan, [grads[i] for i in need], 1)))
        return (None, None, None, *(back.get(i) for i in range(len(grads))))


def apply_rotary(tensors, positions, freqs, *, pairs=None, layout="interleaved", magnitude=1.0):
    """Queries and keys turned to their positions: one tensor [batch, heads, tokens,
    head_dim] or a sequence of up to four alike but for their heads (any strides with
    contiguous channels, such as views of the projections); a tensor or a tuple comes
    back, dense, with tokens and heads in memory in the order of the input's.

    positions: int32 or int64 [tokens] or [batch, tokens]; for several axes of
    coordinates [..., tokens, axes] with ``pairs`` giving each axis its share of the
    pairs.  freqs: float64 [P], radians a position, on the device; 2P channels of a
    head turn, channels 2j and 2j + 1 (interleaved) or j and P + j (half), and are
    multiplied by magnitude; the rest are copied.  Angles are formed in 64 bits.
    Differentiable in the tensors (first order)."""
    one = isinstance(tensors, torch.Tensor)
    tensors = (tensors,) if one else tuple(tensors)
    plan, freqs = _plan(tensors, positions, freqs, pairs, layout, float(magnitude))
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        outs = _Rotary.apply(plan, positions, freqs, *tensors)
    else:
        outs = _turn(plan, tensors, 0)
    return outs[0] if one else outs


@dataclass(frozen=True)
class RotaryEncoding:
    """How ``PACK3DAttention(rotary=...)`` turns q, kl and kg: the coordinates (or, with
    position_encoding="packed", the packed rows) as positions, ``fraction`` of each
    head's pairs turned, layout and scaling as in apply_rotary and
    rotary_frequencies (trained: positions an axis had in training)."""

    layout: str = "interleaved"
    fraction: float = 1.0
    base: float = 10000.0
    scaling: str = "none"
    factor: float = 1.0
    trained: float | None = None

    def __post_init__(self):
        if self.layout not in LAYOUTS:
            raise ValueError("layout must be interleaved or half")
        if not 0.0 < self.fraction <= 1.0:
            raise ValueError("fraction must be in (0, 1]")
        rotary_frequencies(1, base=self.base, scaling=self.scaling, factor=self.factor, trained=self.trained)

    def pairs(self, head_dim, axes):
        total = max(axes, int(head_dim // 2 * self.fraction))
        return tuple(total // axes + (a < total % axes) for a in range(axes))

    def frequencies(self, head_dim, axes, device):
        """(pairs, frequencies on the device, magnitude)."""
        pairs = self.pairs(head_dim, axes)

        def make():
            freqs, magnitude = rotary_frequencies(pairs, base=self.base, scaling=self.scaling, factor=self.factor,
                                                  trained=self.trained)
            return freqs.to(device), magnitude
        return (pairs, *_cached(("rotary", self, pairs, str(device)), make))
