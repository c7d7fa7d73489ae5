"""Causal softmax attention with grouped heads on MI355X, for the layers that hybrid stacks put between the delta-rule ones
(the reference's ``CausalSelfAttention``, modules/attention/causal.py:99, is the same function behind its projections).

``causal_attention(q, k, v, scale=None, *, cu_seqlens=None)`` takes ``q [B,H,T,d]`` and ``k, v [B,Hkv,T,d]`` with H a multiple of
Hkv (query head h reads key head ``h // (H // Hkv)``), float32 or bfloat16, d at most 128, and returns ``o`` in q's dtype and memory
order: ``[B,T,H,d]`` tensors are passed as ``x.transpose(1, 2)`` views and nothing is copied.  Packed batches pass B = 1 and
``cu_seqlens``, like the chunked ops; no query sees another sequence.  Differentiable with respect to q, k and v.
``causal_attention_step(q, k, v, k_cache, v_cache, lengths, scale=None)`` is one decode token: its key and value are written into the
caches at ``lengths`` and its queries attend to everything up to it.  There is no other code path: the ops raise if the library is
missing.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .linear_attn import _check_cu_seqlens

Tensor = torch.Tensor


def causal_attention(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None, *, cu_seqlens=None) -> Tensor:
    """``softmax(scale q k^T + causal mask) v``; ``scale`` defaults to ``d ** -0.5``."""
    cu = None
    if cu_seqlens is not None:
        cu = _check_cu_seqlens(cu_seqlens, q.shape[2]).to(device=q.device, dtype=torch.int32).contiguous()
    return _lib.host().causal_attention(q, k, v, scale, cu)


def causal_attention_step(q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, scale: Optional[float] = None) -> Tensor:
    """One token per sequence: ``q [B,H,d]``, ``k, v [B,Hkv,d]``, caches ``[B,Hkv,S,d]`` (d a multiple of 8; strided views are fine, they
    are written in place), ``lengths [B]`` int32 on the GPU: tokens each sequence already holds.  Returns ``o [B,H,d]``.  The caller
    advances ``lengths``.  Places behind the token are not read; a length outside ``0 .. S - 1`` writes nothing and gives NaN."""
    return _lib.host().causal_attention_step(q, k, v, k_cache, v_cache, lengths, scale)
