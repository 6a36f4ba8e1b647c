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

from . import _lib
from .rope import _cached

LAYOUTS = ("interleaved", "half")
SCALINGS = ("none", "linear", "ntk", "parts")


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
    if layout not in LAYOUTS:
        raise ValueError("layout must be interleaved or half")
    one = isinstance(tensors, torch.Tensor)
    outs = _lib.ops().rotary([tensors] if one else tensors, positions, freqs, pairs, layout == "half", magnitude)
    return outs[0] if one else tuple(outs)


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
