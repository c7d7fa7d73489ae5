"""Element-wise gated linear recurrence on MI355X: the mixer of layers whose state is one number per channel, next to the
delta-rule scans, whose state is a matrix per head.

``gated_linear_recurrence(x, g, initial_state=None, *, cu_seqlens=None)`` computes ``h_t = exp(g_t) * h_{t-1} + x_t`` over
``x, g [B,T,D]`` and returns ``(y, final_state)``: ``y = h`` in x's dtype, the state ``[B,D]`` in float32.  ``g`` holds log-decays
(<= 0; -inf drops everything before the token) in float32 or in x's dtype; x and g may be strided views over batch and time
(slices of one projection).  Packed batches pass ``x [1,T,D]`` with ``cu_seqlens`` and states ``[nseq,D]``, like the chunked ops.
Differentiable with respect to x, g and the initial state; the states between the passes are float32 whatever x is.
``gated_linear_recurrence_step(x, g, state, *, inplace=False)`` is one decode token on ``[B,D]`` tensors, in place on request
(not differentiable then).  There is no other code path: the ops raise if the library is missing.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .linear_attn import _check_cu_seqlens

Tensor = torch.Tensor


def gated_linear_recurrence(x: Tensor, g: Tensor, initial_state: Optional[Tensor] = None, *, cu_seqlens=None) -> Tuple[Tensor, Tensor]:
    """``h_t = exp(g_t) h_{t-1} + x_t`` over ``[B,T,D]``; returns ``(h in x's dtype, last h in float32)``."""
    cu = None
    if cu_seqlens is not None:
        cu = _check_cu_seqlens(cu_seqlens, x.shape[1]).to(device=x.device, dtype=torch.int32).contiguous()
    return _lib.host().linrec(x, g, initial_state, cu)


def gated_linear_recurrence_step(x: Tensor, g: Tensor, state: Tensor, *, inplace: bool = False) -> Tuple[Tensor, Tensor]:
    """One token of the recurrence: ``x, g, state [B,D]``; returns ``(h in x's dtype, h in float32)``."""
    return _lib.host().linrec_step(x, g, state, inplace)
