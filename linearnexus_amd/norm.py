"""Gated RMSNorm output epilogue on MI355X: ``rmsnorm_gated(x, gate, weight, eps)`` computes what the reference's
``FusedRMSNormGated`` module does in its ``__call__`` (linearnexus/modules/linear_attn/kda.py:664-700):
``RMSNorm(x) * weight * sigmoid(gate)`` over the last dimension; ``gate=None`` gives the plain RMSNorm the blocks
use without an output gate (gated_deltanet.py:861-862).  Differentiable with respect to x, gate and weight through
the HIP backward kernel.

``rmsnorm_residual(x, residual, weight, post_weight, gate, scale, eps)`` is what stands between two blocks of a stack: the norm
behind a block with its gate and residual scale, the addition to the residual stream and the norm before the next block (the
reference's blocks add and norm separately, modules/common.py:27, kda.py:831-995), one pass forward and one backward.

``layer_norm(x, weight, bias, eps)`` is the norm with a mean, for blocks and heads that take one (the reference's ``LayerNorm``, modules/common.py): weights
for the last dimension, or a set for each head.

There is no other code path: the ops raise if the library is missing.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

Tensor = torch.Tensor


def rmsnorm_gated(x: Tensor, gate: Optional[Tensor], weight: Tensor, eps: float = 1e-5) -> Tensor:
    """``x * rsqrt(mean(x^2, -1) + eps) * weight * sigmoid(gate)`` (kda.py:683-700); ``x, gate [..., d]``, ``weight [d]``."""
    return _lib.host().rmsnorm_gated(x, gate, weight, eps)


def rmsnorm_residual(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], post_weight: Optional[Tensor] = None,
                     gate: Optional[Tensor] = None, scale: Union[float, Tensor] = 1.0, eps: float = 1e-5) -> Tuple[Optional[Tensor], Tensor]:
    """``u = RMSNorm(x) * post_weight * sigmoid(gate)``, ``r = residual + scale * u``, ``z = RMSNorm(r) * weight``; returns ``(z, r)``.

    Norms are over the last dimension (at most 8192 wide).  ``post_weight=None``: x itself takes the place of its norm; ``gate=None``: no
    gate; ``residual=None``: ``r = scale * u`` (the first block); ``weight=None``: z is None (behind the last block).  ``scale`` is a number
    or a ``[d]`` tensor.  ``x [..., d]`` and z are float32 or bfloat16, the residual and r float32 or x's dtype, the gate likewise (one of
    another type is taken in float32); z is the norm of the sum before it is rounded to r's dtype.  Differentiable with respect to every tensor."""
    return _lib.host().rmsnorm_residual(x, residual, weight, post_weight, gate, scale, eps)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) * rsqrt(var + eps) * weight + bias`` over the last dimension (at most 8192 wide), ``var`` the mean of the squared differences.

    ``x [..., d]`` and the result are float32 or bfloat16; sums are float32.  ``weight`` and ``bias`` are ``[d]``, or ``[heads, d]`` for
    ``x [..., heads, d]``: every head is a row of its own with its own weights (the norm behind a linear-attention mixer).  ``None``: ones, zeros.
    Differentiable with respect to all three, once: asking for a second derivative raises."""
    return _lib.host().layer_norm(x, weight, bias, eps)
