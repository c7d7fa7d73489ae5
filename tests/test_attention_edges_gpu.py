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


# -- dimensions of one element, whose strides say nothing ----------------------------------------------------------

def _slices(B, T, H, Hkv, d, dtype, more):
    """q, k, v as a fused projection leaves them, its rows `more` columns longer than what the heads take."""
    width = (H + 2 * Hkv) * d + more
    g = torch.Generator().manual_seed(3)
    p = torch.randn(B, T, width, generator=g).to(DEV, torch.bfloat16 if dtype == "bf16" else torch.float32)
    cut = lambda first, h: p.as_strided((B, T, h, d), (T * width, width, d, 1), first)
    return cut(0, H), cut(H * d, Hkv), cut((H + Hkv) * d, Hkv)


@pytest.mark.parametrize("dtype,more", [("bf16", 4), ("f32", 2)])
@pytest.mark.parametrize("B,T,H,Hkv", [(1, 1, 4, 1), (1, 1, 2, 2), (3, 1, 4, 1), (1, 5, 4, 1), (1, 5, 1, 1)])
def test_prompt_strides_of_single_elements(B, T, H, Hkv, dtype, more):
    q, k, v = (t.transpose(1, 2) for t in _slices(B, T, H, Hkv, 64, dtype, more))
    do = _slices(B, T, H, Hkv, 64, dtype, more)[0].transpose(1, 2)
    _check(q, k, v, do)


@pytest.mark.parametrize("dtype,more", [("bf16", 4), ("f32", 2)])
@pytest.mark.parametrize("B,H,Hkv", [(1, 8, 1), (1, 4, 2), (2, 4, 1)])
def test_step_strides_of_single_elements(B, H, Hkv, dtype, more):
    q, k, v = (t[:, 0] for t in _slices(B, 1, H, Hkv, 64, dtype, more))
    _, _, _, kc, vc = _step_inputs(B, H, Hkv, 50, 64, dtype)
    _check_step(q, k, v, kc, vc, [49 - b for b in range(B)])


@pytest.mark.parametrize("dtype,more", [("bf16", 4), ("f32", 2)])
@pytest.mark.parametrize("Hkv,S", [(1, 40), (2, 1), (1, 1)])
def test_step_cache_strides_of_single_elements(Hkv, S, dtype, more):
    """Caches of one sequence (and one key head, one place) inside a buffer whose rows the strides of those dimensions do not fit."""
    q, k, v, kc, vc = _step_inputs(1, 4, Hkv, S, 64, dtype)

    def odd(t):
        strides = [64 * Hkv * S + more, 64 * S + (more if Hkv == 1 else 0), 64 + (more if S == 1 else 0), 1]
        return torch.empty(t.numel() + 64, device=DEV, dtype=t.dtype).as_strided(t.shape, strides).copy_(t)

    _check_step(q, k, v, odd(kc), odd(vc), [S - 1])


# -- packed batches of short and long documents ---------------------------------------------------------------------

@pytest.mark.parametrize("lens,H,Hkv,d", [([3, 300], 4, 2, 64), ([1, 2, 500], 8, 4, 64), ([2, 700, 5], 2, 1, 128), ([7, 0, 400, 1, 128], 4, 2, 80)], ids=str)
def test_short_documents_beside_long_ones_are_as_exact_as_their_rounding(lens, H, Hkv, d):
    """A document's operands go in in two parts by its own length, whatever it is packed with."""
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, do = _inputs(1, H, Hkv, cu[-1], d, "bf16")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = la.causal_attention(*leaves, cu_seqlens=cu)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    G = H // Hkv
    nq, nk, nv, nd = (_np(t[0]) for t in (q, k, v, do))
    for lo, hi in zip(cu[:-1], cu[1:]):
        if not 0 < hi - lo <= 128:
            continue
        for kv in range(Hkv):
            sums = {"dk": (0, 0), "dv": (0, 0)}
            for h in range(kv * G, (kv + 1) * G):
                ref = _reference(nq[h, lo:hi], nk[kv, lo:hi], nv[kv, lo:hi], nd[h, lo:hi], d ** -0.5, 2.0 ** -16)
                _within(o[0, h, lo:hi], *ref["o"], f"o {lo}")
                _within(dq[0, h, lo:hi], *ref["dq"], f"dq {lo}")
                sums = {n: (sums[n][0] + ref[n][0], sums[n][1] + ref[n][1] + G * UP * ref[n][0].abs()) for n in sums}
            _within(dk[0, kv, lo:hi], *sums["dk"], f"dk {lo}")
            _within(dv[0, kv, lo:hi], *sums["dv"], f"dv {lo}")
    _check(q, k, v, do, cu=cu)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("lens", [[100], [100, 300, 3, 128]], ids=str)
def test_values_behind_the_mask_of_short_documents(lens, d, bad):
    """Keys and values behind a row's queries, and queries and gradients before a key, are not in its results, in either form of the kernels."""
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, do = _inputs(1, 4, 2, cu[-1], d, "bf16")
    cut = 57  # of the first document
    keep = do.clone()
    keep[:, :, cut:100] = 0

    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = la.causal_attention(*leaves, cu_seqlens=cu)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    clean = run(q, k, v, keep)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, cut:100] = bad
    v2[:, :, cut:100] = bad
    dirty = run(q, k2, v2, keep)
    rest = torch.tensor([i for i in range(cu[-1]) if not cut <= i < 100], device=DEV)
    for a, b in zip(dirty[:2], clean[:2]):
        assert torch.equal(a[:, :, rest], b[:, :, rest])
    assert not bool(torch.isfinite(dirty[0][:, :, cut:100]).any())
    q2, do2 = q.clone(), do.clone()
    q2[:, :, :20] = bad
    do2[:, :, :20] = bad
    full, dirty = run(q, k, v, do), run(q2, k, v, do2)
    for a, b in zip(dirty[2:], full[2:]):
        assert torch.equal(a[:, :, 20:], b[:, :, 20:])


def test_packed_documents_of_both_kinds_in_a_replayed_graph():
    q, k, v, do = _inputs(1, 4, 2, 640, 128, "bf16", token_first=True)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    cu = torch.tensor([0, 3, 303, 303, 400, 640], dtype=torch.int32, device=DEV)

    def both():
        o = la.causal_attention(*leaves, cu_seqlens=cu)
        return (o, *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for table in ([0, 3, 303, 303, 400, 640], [0, 1, 2, 3, 4, 640], [0, 128, 256, 384, 512, 640], [0, 129, 258, 387, 516, 640]):
        cu.copy_(torch.tensor(table, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both()))


# -- memory order ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [20, 33, 64, 80])
@pytest.mark.parametrize("how", ["head first", "token first", "slice of a projection"])
def test_results_lie_as_the_queries_do(how, d):
    B, T, H = 2, 9, 4
    q, k, v, do = _inputs(B, H, 2, T, d, "bf16", token_first=how != "head first")
    if how == "slice of a projection":
        q = torch.cat([q.transpose(1, 2).flatten(2), torch.zeros(B, T, 48, device=DEV, dtype=q.dtype)], 2)[..., : H * d].unflatten(2, (H, d)).transpose(1, 2)
    with torch.no_grad():
        o = la.causal_attention(q, k, v)
    leaf = q.detach().requires_grad_()
    graded = la.causal_attention(leaf, k, v)
    for t in (o, graded):
        assert (t if how == "head first" else t.transpose(1, 2)).is_contiguous() and torch.equal(t, o)
    _check(q, k, v, do)
