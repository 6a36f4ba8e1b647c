"""Dropout from a counter-based generator: the mask is a function of a seed, an
offset and the element's index, computed where it is needed and never stored.

``counter_dropout`` applies it to a tensor; ``block.block_residual`` applies the
same mask inside the end of a block.  Element i of a tensor in row-major order
compares 16 bits of Philox4x32-10 (Salmon et al., 2011) for the counter
(i // 8, offset) and the key seed with round(65536 p), so the rate is a multiple
of 2^-16; what is kept is divided by the share that this rate keeps.
"""
from __future__ import annotations

import torch

from . import _lib


def threshold_of(p):
    """The 16-bit threshold of rate p."""
    if not 0.0 <= p < 1.0:
        raise ValueError("dropout rate must be in [0, 1)")
    return min(65535, int(p * 65536 + 0.5))


def new_seed(device):
    """A seed tensor (seed, offset) from torch's generator of the device; under
    graph capture each replay draws another."""
    return torch.randint(0, 2 ** 62, (2,), dtype=torch.int64, device=device)


def mask_args(p, seed, device):
    """(threshold, seed tensor or None, seed, offset) of rate p.  seed: an int, a pair of ints
    (seed, offset), or an int64 tensor of these two on the device, which the kernels read
    (no host synchronisation)."""
    threshold = threshold_of(p)
    if not threshold:
        return 0, None, 0, 0
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,) or seed.device != device:
            raise ValueError("a seed tensor must be int64 [2] (seed, offset) on the input's device")
        return threshold, seed if seed.stride(0) == 1 else seed.contiguous(), 0, 0
    pair = (seed, 0) if type(seed) is int else seed
    if not (isinstance(pair, (tuple, list)) and len(pair) == 2 and all(type(v) is int and 0 <= v < 2 ** 63
                                                                     for v in pair)):
        raise ValueError("dropout needs a seed: an int, a pair (seed, offset), both in [0, 2^63), or an int64 tensor [2]")
    return threshold, None, *pair


def counter_dropout(x, p, seed):
    """x with each element dropped at rate p (a multiple of 2^-16, the nearest) and the
    others divided by 1 - p.  The same seed gives the same mask, in the backward too;
    another call needs another seed or offset.  fp32, fp16 and bf16, any shape (a
    tensor that is not contiguous is copied first); differentiable (first order).
    A rate that rounds to 0 gives x itself."""
    mask = mask_args(p, seed, x.device)
    if not mask[0] and x.is_cuda and x.dtype in _lib.DTYPES:
        return x
    return _lib.ops().dropout(x, *mask)
