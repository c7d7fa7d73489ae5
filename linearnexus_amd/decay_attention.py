"""Linear attention with a decay for each head on MI355X: the mixer whose state is a matrix per head that fades and grows, without the delta rule's
erasing (the scans of linear_attn.py), for prompts, training and decoding.

``decay_linear_attention(q, k, v, g, scale=None, initial_state=None, *, cu_seqlens=None)`` computes ``S_t = exp(g_t) S_{t-1} + k_t^T v_t`` and
``o_t = scale q_t S_t`` over ``q, k [B,H,T,dk]`` and ``v [B,H,T,dv]`` (float32 or bfloat16, dk and dv at most 256) and returns ``(o, final_state)``:
o in q's dtype and memory order, the state ``[B,H,dk,dv]`` in float32.  ``[B,T,H,d]`` tensors are passed as ``x.transpose(1, 2)`` views and nothing is
copied.  ``g`` holds log-decays (<= 0; -inf drops everything before the token): ``[B,H,T]``, any strides, or one constant for each head, ``[H]``.
Packed batches pass B = 1, ``cu_seqlens`` and states ``[nseq,H,dk,dv]``, like the chunked ops.  Differentiable with respect to q, k, v, g and the
initial state, once: asking for a second derivative raises; states and sums are float32 whatever q is.
``decay_linear_attention_step(q, k, v, g, state, scale=None, *, inplace=False)`` is one decode token on ``[B,H,d]`` tensors, in place on request (not
differentiable then).  There is no other code path: the ops raise if the library is missing.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .linear_attn import _check_cu_seqlens

Tensor = torch.Tensor


def decay_linear_attention(q: Tensor, k: Tensor, v: Tensor, g: Tensor, scale: Optional[float] = None, initial_state: Optional[Tensor] = None, *,
                           cu_seqlens=None) -> Tuple[Tensor, Tensor]:
    """``S_t = exp(g_t) S_{t-1} + k_t^T v_t``, ``o_t = scale q_t S_t``; returns ``(o in q's dtype, last S in float32)``; ``scale`` defaults to ``dk ** -0.5``."""
    cu = None
    if cu_seqlens is not None:
        cu = _check_cu_seqlens(cu_seqlens, q.shape[2]).to(device=q.device, dtype=torch.int32).contiguous()
    return _lib.host().decay_attention(q, k, v, g, scale, initial_state, cu)


def decay_linear_attention_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, state: Tensor, scale: Optional[float] = None, *,
                                inplace: bool = False) -> Tuple[Tensor, Tensor]:
    """One token: ``q, k [B,H,dk]``, ``v [B,H,dv]``, ``g [B,H]`` or ``[H]``, ``state [B,H,dk,dv]``; returns ``(o [B,H,dv], S in float32)``."""
    return _lib.host().decay_attention_step(q, k, v, g, state, scale, inplace)
