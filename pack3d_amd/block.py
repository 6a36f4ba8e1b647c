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

from typing import NamedTuple, Optional

import torch

from . import _lib
from .dropout import mask_args

KINDS = {"layer": 1, "rms": 2}  # enum p3d_norm_kind


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


def _norm_args(name, norm):
    """(kind, weight, bias, eps) for the binding."""
    if norm is None:
        return 0, None, None, 0.0
    if not isinstance(norm, Norm) or norm.kind not in KINDS:
        raise ValueError(f"{name} must be a Norm of kind layer or rms")
    return KINDS[norm.kind], norm.weight, norm.bias, norm.eps


_NO_NORM, _NO_MASK = (0, None, None, 0.0), (0, None, 0, 0)


def block_norm(x, norm: Norm, *, dtype=None):
    """``norm`` of x [batch, tokens, dim] or [tokens, dim] in ``dtype`` (x's own; for an
    fp32 x also fp16 or bf16, as the next products take it): statistics in fp32, one
    rounding, any row stride.  Differentiable in x and the norm's parameters."""
    if norm is None:
        raise ValueError("block_norm needs a Norm")
    return _lib.ops().block(x, None, None, None, *_NO_NORM, *_norm_args("norm", norm), 1.0, *_NO_MASK, dtype)


def block_residual(x, y, *, post_norm: Optional[Norm] = None, gate=None, scale=None, alpha=1.0, p=0.0, seed=None,
                   next_norm: Optional[Norm] = None):
    """The end of a block: ``alpha * x + scale * gate * dropout(post_norm(y))``, and with
    ``next_norm`` the pair of that sum and its norm, from one pass over the rows.

    x, y: [batch, tokens, dim] or [tokens, dim]; y has x's type or, over an fp32 x, fp16
    or bf16.  The sum has x's type, the norm y's (computed from the unrounded sum).
    gate: [batch or 1, 1, dim] (per sample), [batch, tokens, 1] or [batch, tokens, dim].
    scale: [dim], per channel.  p, seed: as counter_dropout's, on y's elements.
    Differentiable in x, y, gate, scale and the norms' parameters (first order)."""
    return _lib.ops().block(x, y, gate, scale, *_norm_args("post_norm", post_norm), *_norm_args("next_norm", next_norm),
                            alpha, *(mask_args(p, seed, x.device) if p != 0.0 else _NO_MASK), None)
