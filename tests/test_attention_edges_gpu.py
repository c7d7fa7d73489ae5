"""Causal attention at its edges, with the float64 definition and the elementwise bounds of test_attention_gpu."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la
from test_attention_gpu import DEV, U, UP, _check, _check_step, _inputs, _np, _reference, _step_inputs, _within

pytestmark = pytest.mark.gpu


# -- one token: the weights enter the product in two bfloat16 parts ------------------------------------------------

@pytest.mark.parametrize("B,H,Hkv,S,d,lens", [(1, 4, 1, 40, 64, [39]), (2, 8, 8, 300, 80, [64, 299]), (2, 16, 4, 1000, 128, [999, 511]), (1, 8, 2, 3000, 128, [2700]),
                                              (1, 40, 1, 700, 40, [640])])
def test_step_is_as_exact_as_its_rounding(B, H, Hkv, S, d, lens):
    """A weight is rounded by 2^-8 of itself and what that left by 2^-8 of that: 2^-16 is what the two parts are off by."""
    q, k, v, kc, vc = _step_inputs(B, H, Hkv, S, d, "bf16")
    o = la.causal_attention_step(q, k, v, kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV))
    s, r = d ** -0.5, 2.0 ** -16
    for b, n in enumerate(lens):
        for h in range(H):
            key, val, query = _np(kc[b, h * Hkv // H, : n + 1]), _np(vc[b, h * Hkv // H, : n + 1]), _np(q[b, h])
            S_ = key @ query * s
            ES = (d + 8) * UP * s * (key.abs() @ query.abs()) + 4 * U * S_.abs()
            P = torch.softmax(S_, 0)
            EP = P * (ES + 2 * ES.max() + (n + 32) * UP)
            _within(o[b, h], P @ val, (EP + (r + (n + 32) * UP) * P) @ val.abs(), f"o {b} {h}")
