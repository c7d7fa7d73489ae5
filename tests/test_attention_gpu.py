"""Causal attention against its definition in float64, with elementwise bounds.

Bounds.  r = 2^-8 where an operand is rounded to bfloat16 and 0 in float32, u = 2^-24; a matrix product adds up in float32, two units
per addition (u' = 2^-23).  With S = scale q k^T, |S|* = |scale| |q| |k|^T and T keys:
  E_S = (d + 8) u' |S|* + 4 u |S|       a score's sum, its scaling and the exponential's argument
  P: relative E_S + max over the row of E_S (the reference or the logarithm of the sum) + (T + 16) u' (the row's sum)
  o: r P |v| (the rounded operand) + E_P |v| + (T + 16) u' P |v|
  dP = do v^T: (d + 8) u' |do| |v|^T;  delta = o . do: r |o| |do| + E_o |do| + d u' |o| |do| (o is read back as it was rounded)
  dS = P (dP - delta): E_P |dP - delta| + P (E_dP + E_delta), and r |dS| as an operand
  dq = scale dS k, dk = scale dS^T q, dv = P^T do: the operands' bounds times the magnitudes, (T + 16) u' for the sum
and every output is rounded once, eps / 2 of its value.  Second-order terms are covered by a factor of 1.1."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, UP = 2.0 ** -24, 2.0 ** -23
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _np(t):
    return t.detach().double().cpu()


def _reference(q, k, v, do, scale, r):
    """One sequence and head in float64: values and bounds of o, dq, dk, dv."""
    T, d = q.shape
    hide = torch.ones(T, T, dtype=torch.bool).triu(1)
    S = (q @ k.T * scale).masked_fill(hide, -np.inf)
    P = torch.softmax(S, 1)
    mag = abs(scale) * (q.abs() @ k.abs().T)
    ES = (d + 8) * UP * mag + 4 * U * (q @ k.T * scale).abs()
    ES = ES.masked_fill(hide, 0)
    EP = P * (ES + ES.amax(1, True) + (T + 16) * UP)
    o = P @ v
    Eo = (EP + (r + (T + 16) * UP) * P) @ v.abs()
    out = {"o": (o, Eo)}
    if do is None:
        return out
    dP = do @ v.T
    EdP = (d + 8) * UP * (do.abs() @ v.abs().T)
    delta = (o * do).sum(1, True)
    Ed = ((r + d * UP) * (o.abs() * do.abs()) + Eo * do.abs()).sum(1, True)
    diff = (dP - delta).masked_fill(hide, 0)
    dS = P * diff
    EdS = EP * diff.abs() + P * (EdP + Ed) + (r + (T + 16) * UP) * dS.abs()
    a = abs(scale)
    out["dq"] = (scale * dS @ k, a * EdS @ k.abs())
    out["dk"] = (scale * dS.T @ q, a * EdS.T @ q.abs())
    out["dv"] = (P.T @ do, (EP + (r + (T + 16) * UP) * P).T @ do.abs())
    return out


def _within(got, ref, bound, what):
    eps = torch.finfo(got.dtype).eps / 2
    g = _np(got)
    tol = 1.1 * bound + eps * (ref.abs() + bound) + 1e-36
    worst = ((g - ref).abs() / tol).nan_to_num(nan=np.inf)
    assert g.shape == ref.shape and float(worst.max() if worst.numel() else 0) <= 1, f"{what}: {float(worst.max()):.2f} of the bound"


def _inputs(B, H, Hkv, T, d, dtype, token_first=False, seed=0):
    g = torch.Generator().manual_seed(seed)

    def n(h, std=1.0):
        x = (torch.randn(B, T, h, d, generator=g) * std).to(DEV, DT[dtype])
        return x.transpose(1, 2) if token_first else x.transpose(1, 2).contiguous()

    return n(H, 1.5), n(Hkv), n(Hkv), n(H)


def _check(q, k, v, do, scale=None, cu=None, r=None):
    B, H, T, d = q.shape
    G = H // k.shape[1]
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = la.causal_attention(*leaves, scale, cu_seqlens=cu)
    assert o.shape == q.shape and o.dtype == q.dtype
    with torch.no_grad():
        assert torch.equal(la.causal_attention(q, k, v, scale, cu_seqlens=cu), o)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    s = d ** -0.5 if scale is None else scale
    if r is None:
        r = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    spans = [(0, T)] if cu is None else list(zip(cu[:-1], cu[1:]))
    nq, nk, nv, nd = (_np(t) for t in (q, k, v, do))
    for b in range(B):
        for lo, hi in spans:
            if lo == hi:
                continue
            for kv in range(H // G):
                sums = {}
                for h in range(kv * G, (kv + 1) * G):
                    ref = _reference(nq[b, h, lo:hi], nk[b, kv, lo:hi], nv[b, kv, lo:hi], nd[b, h, lo:hi], s, r)
                    _within(o[b, h, lo:hi], *ref["o"], "o")
                    _within(dq[b, h, lo:hi], *ref["dq"], "dq")
                    for name in ("dk", "dv"):
                        val, bound = sums.get(name, (0, 0))
                        sums[name] = (val + ref[name][0], bound + ref[name][1] + G * UP * ref[name][0].abs())
                _within(dk[b, kv, lo:hi], *sums["dk"], "dk")
                _within(dv[b, kv, lo:hi], *sums["dv"], "dv")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,Hkv,T,d", [(1, 1, 1, 1, 8), (2, 2, 1, 2, 64), (1, 4, 2, 31, 64), (2, 3, 3, 32, 40), (1, 2, 1, 33, 128), (1, 2, 2, 63, 80),
                                         (2, 2, 1, 64, 128), (1, 6, 2, 65, 72), (1, 2, 1, 127, 128), (1, 8, 8, 128, 64), (1, 2, 1, 129, 16), (2, 4, 1, 257, 128),
                                         (1, 2, 1, 100, 33), (2, 8, 4, 200, 128), (1, 8, 1, 385, 128), (1, 2, 1, 700, 64)])
def test_forward_and_gradients(B, H, Hkv, T, d, dtype):
    _check(*_inputs(B, H, Hkv, T, d, dtype, token_first=T % 2 == 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,d", [(2, 1, 64), (8, 8, 128)])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [0, 5, 0, 0, 200, 1, 0], [64, 128, 63, 129, 65], [300, 3, 2]], ids=str)
def test_packed(lens, H, Hkv, d, dtype):
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    _check(*_inputs(1, H, Hkv, cu[-1], d, dtype, token_first=True), cu=cu)


def test_many_short_sequences():
    cu = list(range(0, 3 * 150 + 1, 3))  # more than a wave of sequences
    _check(*_inputs(1, 2, 1, 450, 64, "bf16"), cu=cu)


@pytest.mark.parametrize("lens,H,Hkv,d", [([1], 2, 1, 64), ([2], 8, 4, 64), ([3], 8, 4, 64), ([7], 2, 2, 128), ([64], 2, 1, 128), ([3, 1, 90, 0, 5], 4, 2, 80)], ids=str)
def test_short_sequences_are_as_exact_as_their_rounding(lens, H, Hkv, d):
    """With one tile of keys on average operands go in in two bfloat16 parts: each rounding of 2^-8 is one of 2^-16.  o and what its rounding
    left are bfloat16 each, so delta's is 2^-16, too."""
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    _check(*_inputs(1, H, Hkv, cu[-1], d, "bf16"), cu=cu, r=2.0 ** -16)


def test_more_sequences_than_a_wave_looks_at():
    lens = [0, 3, 1, 0, 70, 2, 0, 1] * 60 + [200]
    _check(*_inputs(1, 2, 1, sum(lens), 16, "bf16"), cu=np.concatenate([[0], np.cumsum(lens)]).tolist())
    cu = np.concatenate([[0], np.cumsum([1, 0, 1] * 1700)]).tolist()  # every query has one key
    q, k, v, do = _inputs(1, 2, 2, cu[-1], 16, "f32")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = la.causal_attention(*leaves, cu_seqlens=cu)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    # the bounds above with T = 1 and P = 1: the weight is exp(S - lse), whose argument is rounded, not 1 itself
    nq, nk, nv, nd = (_np(t) for t in (q, k, v, do))
    mag = 0.25 * (nq.abs() * nk.abs()).sum(-1, True)
    EP = 2 * ((16 + 8) * UP * mag + 4 * U * (0.25 * (nq * nk).sum(-1, True)).abs()) + 17 * UP
    _within(o, nv, (EP + 17 * UP) * nv.abs(), "o")
    _within(dv, nd, (EP + 17 * UP) * nd.abs(), "dv")
    # do . v - delta is the same sum twice: 2 (d + 8) 2^-23 abs(do) . abs(v) (< 40), times scale = 1/4 and abs(k), abs(q) (< 8)
    assert float(dq.abs().max()) < 4.6e-4 and float(dk.abs().max()) < 4.6e-4


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_and_broadcast_heads(dtype):
    q, k, v, do = _inputs(2, 4, 4, 90, 64, dtype)
    fused = torch.cat([q, k, v], 3)  # rows inside rows of a projection
    one = k[:, :1].expand(-1, 4, -1, -1)
    _check(fused[..., :64], fused[..., 64:128], fused[..., 128:], do)
    _check(q, one, v, do)
    _check(q, k, v, do[:, :, :1].expand(-1, -1, 90, -1))
    odd = torch.empty(2 * 4 * 90 * 64 + 1, device=DEV, dtype=q.dtype)[1:].view(2, 4, 90, 64).copy_(q)
    _check(odd, k.transpose(2, 3).contiguous().transpose(2, 3), v, do)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_scales(scale, dtype):
    _check(*_inputs(1, 2, 1, 150, 64, dtype), scale=scale)


def test_large_scores_stay_finite():
    """Scores of many thousands: one key per row has all the weight (float32 products of small integers are exact)."""
    q, k, v, do = (torch.round(3 * t) for t in _inputs(1, 2, 1, 200, 64, "f32"))
    o = la.causal_attention(q, k, v, 100.0)
    S = (_np(q)[0, 1] @ _np(k)[0, 0].T * 100).masked_fill(torch.ones(200, 200, dtype=torch.bool).triu(1), -np.inf)
    assert torch.allclose(_np(o)[0, 1], torch.softmax(S, 1) @ _np(v)[0, 0], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_behind_the_mask_do_not_matter(bad, dtype):
    """Keys and values that no query of a row may see (a padded end) are not in its results, whatever they hold; nor are queries and
    output gradients that come before a key."""
    q, k, v, do = _inputs(1, 4, 2, 150, 128, dtype)
    clean = [t.detach().requires_grad_() for t in (q, k, v)]
    o = la.causal_attention(*clean)
    keep = do.clone()
    keep[:, :, 77:] = 0
    want = torch.autograd.grad(o, clean, keep)
    dirty = [t.detach().clone() for t in (q, k, v)]
    dirty[1][:, :, 77:] = bad
    dirty[2][:, :, 77:] = bad
    leaves = [t.requires_grad_() for t in dirty]
    o2 = la.causal_attention(*leaves)
    eps = torch.finfo(q.dtype).eps
    assert torch.allclose(o2[:, :, :77].float(), o[:, :, :77].float(), rtol=2 * eps, atol=2 * eps)
    dq = torch.autograd.grad(o2, leaves, keep)[0]
    assert torch.allclose(dq[:, :, :77].float(), want[0][:, :, :77].float(), rtol=8 * eps, atol=8 * eps)
    assert not bool(torch.isfinite(o2[:, :, 77:]).any())
    first = q.clone()
    first[:, :, :20] = bad  # the first queries: they see keys 0 .. 19 only
    leaves = [t.detach().requires_grad_() for t in (first, k, v)]
    gq, gk, gv = torch.autograd.grad(la.causal_attention(*leaves), leaves, do)
    full = torch.autograd.grad(la.causal_attention(*clean), clean, do)
    for got, ref in ((gk, full[1]), (gv, full[2])):
        assert torch.allclose(got[:, :, 20:].float(), ref[:, :, 20:].float(), rtol=8 * eps, atol=8 * eps)
    lone = do.clone()
    lone[:, :, 3] = bad
    gk, gv = torch.autograd.grad(la.causal_attention(*clean), clean[1:], lone)
    for got, ref in ((gk, full[1]), (gv, full[2])):
        assert torch.allclose(got[:, :, 4:].float(), ref[:, :, 4:].float(), rtol=8 * eps, atol=8 * eps)


def test_packed_sequences_do_not_see_each_other():
    q, k, v, do = _inputs(1, 2, 1, 200, 64, "bf16")
    cu = [0, 70, 200]
    o = la.causal_attention(q, k, v, cu_seqlens=cu)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, :70] = float("nan")
    v2[:, :, :70] = float("nan")
    o2 = la.causal_attention(q, k2, v2, cu_seqlens=torch.tensor(cu, device=DEV))
    assert torch.equal(o2[:, :, 70:], o[:, :, 70:])


def test_gradients_against_differences():
    """Central differences in float32 with steps of 1e-2: the remainder is step^2 of a third derivative of order one."""
    q, k, v, do = _inputs(1, 2, 1, 40, 16, "f32")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    loss = lambda a: (la.causal_attention(*a) * do).double().sum()
    grads = torch.autograd.grad(loss(leaves), leaves)
    g = torch.Generator().manual_seed(2)
    for i in range(3):
        dirn = torch.randn(leaves[i].shape, generator=g).to(DEV)
        up, down = [t.detach().clone() for t in leaves], [t.detach().clone() for t in leaves]
        up[i] += 1e-2 * dirn
        down[i] -= 1e-2 * dirn
        diff = (loss(up) - loss(down)) / 2e-2
        assert abs(float(diff - (grads[i].double() * dirn).sum())) < 1e-2 * float((grads[i].double() * dirn).abs().sum())


def test_repeats_bit_for_bit_and_replays():
    q, k, v, do = _inputs(2, 4, 2, 300, 128, "bf16")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def both():
        o = la.causal_attention(*leaves)
        return (o, *torch.autograd.grad(o, leaves, do))

    assert all(torch.equal(a, b) for a, b in zip(both(), both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(3):
        with torch.no_grad():
            leaves[1].copy_(torch.randn_like(leaves[1]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both()))


# -- one token --------------------------------------------------------------------------------------------------

def _step_inputs(B, H, Hkv, S, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(DEV, DT[dtype])
    return n(B, H, d) * 1.5, n(B, Hkv, d), n(B, Hkv, d), n(B, Hkv, S, d), n(B, Hkv, S, d)


def _check_step(q, k, v, kc, vc, lens, scale=None):
    B, H, d = q.shape
    G = H // k.shape[1]
    k0, v0 = kc.clone(), vc.clone()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = la.causal_attention_step(q, k, v, kc, vc, lengths, scale)
    assert o.shape == q.shape and o.dtype == q.dtype and lengths.tolist() == lens
    for b, n in enumerate(lens):
        k0[b, :, n], v0[b, :, n] = k[b], v[b]
    assert torch.equal(kc.nan_to_num(7.0), k0.nan_to_num(7.0)) and torch.equal(vc.nan_to_num(7.0), v0.nan_to_num(7.0))
    s = d ** -0.5 if scale is None else scale
    r = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    for b, n in enumerate(lens):
        for h in range(H):
            key, val = _np(kc[b, h // G, : n + 1]), _np(vc[b, h // G, : n + 1])
            query = _np(q[b, h])
            S = key @ query * s
            ES = (d + 8) * UP * abs(s) * (key.abs() @ query.abs()) + 4 * U * S.abs()
            P = torch.softmax(S, 0)
            EP = P * (ES + 2 * ES.max() + (n + 32) * UP)  # the reference moves between tiles, waves and splits
            _within(o[b, h], P @ val, (EP + (r + (n + 32) * UP) * P) @ val.abs(), f"o {b} {h}")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,Hkv,S,d,lens", [(1, 1, 1, 1, 8, [0]), (2, 4, 1, 40, 64, [0, 39]), (3, 6, 2, 33, 128, [31, 32, 5]), (2, 8, 8, 300, 80, [64, 299]),
                                              (1, 40, 1, 200, 64, [130]), (2, 16, 4, 1000, 128, [999, 511]), (1, 8, 2, 3000, 128, [2700]), (2, 3, 3, 700, 40, [3, 640])])
def test_step(B, H, Hkv, S, d, lens, dtype):
    q, k, v, kc, vc = _step_inputs(B, H, Hkv, S, d, dtype)
    for b, n in enumerate(lens):  # what lies behind the token is nobody's business
        kc[b, :, n:] = float("nan")
        vc[b, :, n:] = float("nan")
    _check_step(q, k, v, kc, vc, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,S,d,n", [(8, 70_000, 128, 69_999), (3, 70_000, 64, 2), (40, 20_000, 40, 17_003)])
def test_step_in_many_shares(H, S, d, n, dtype):
    """One key head and a long cache: hundreds of workgroups share the sequence, or find nothing of it."""
    _check_step(*_step_inputs(1, H, 1, S, d, dtype), [n])


def test_step_refuses_caches_that_share_memory():
    q, k, v, kc, vc = _step_inputs(2, 4, 2, 20, 64, "bf16")
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    for a, b in ((kc, kc), (kc.as_strided(kc.shape, (0, 64 * 20, 64, 1)), vc), (kc, vc.as_strided(vc.shape, (64 * 40, 64 * 20, 8, 1))),
                 (kc, vc.as_strided(vc.shape, (64 * 20, 64 * 20, 64, 1)))):
        with pytest.raises(RuntimeError, match="memory"):
            la.causal_attention_step(q, k, v, a, b, lengths)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.4, 0.0, 3.0])
def test_step_scales(scale, dtype):
    _check_step(*_step_inputs(2, 4, 2, 150, 64, dtype), [149, 60], scale)


def test_step_strided_caches():
    q, k, v, _, _ = _step_inputs(2, 4, 2, 1, 64, "bf16")
    both = torch.randn(2, 90, 2, 2, 64, device=DEV).bfloat16()  # [B, S, key or value, Hkv, d]
    kc, vc = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    _check_step(q, k, v, kc, vc, [88, 10])


def test_step_without_a_place_gives_nan_and_writes_nothing():
    q, k, v, kc, vc = _step_inputs(3, 4, 2, 20, 64, "bf16")
    k0, v0 = kc.clone(), vc.clone()
    o = la.causal_attention_step(q, k, v, kc, vc, torch.tensor([20, -1, 7], dtype=torch.int32, device=DEV))
    assert bool(torch.isnan(o[:2]).all()) and bool(torch.isfinite(o[2]).all())
    assert torch.equal(kc[:2], k0[:2]) and torch.equal(vc[:2], v0[:2]) and torch.equal(kc[2, :, 7], k[2])


def test_prompt_then_tokens():
    """The cache filled from a prompt, then tokens one by one, in a replayed graph that advances the lengths itself."""
    q, k, v, _ = _inputs(2, 4, 2, 70, 64, "f32")
    whole = la.causal_attention(q, k, v)
    kc, vc = torch.zeros(2, 2, 80, 64, device=DEV), torch.zeros(2, 2, 80, 64, device=DEV)
    kc[:, :, :60], vc[:, :, :60] = k[:, :, :60], v[:, :, :60]
    lengths = torch.full((2,), 60, dtype=torch.int32, device=DEV)
    tok = [t[:, :, 60].clone() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        la.causal_attention_step(*tok, kc, vc, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = la.causal_attention_step(*tok, kc, vc, lengths)
        lengths.add_(1)
    for t in range(60, 70):
        for buf, x in zip(tok, (q, k, v)):
            buf.copy_(x[:, :, t])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(o, whole[:, :, t], rtol=1e-5, atol=1e-5)
    assert torch.equal(kc[:, :, :70], k) and lengths.tolist() == [70, 70]


def test_empty():
    z = torch.zeros(2, 4, 0, 64, device=DEV, requires_grad=True)
    o = la.causal_attention(z, z[:, :2], z[:, :2])
    assert o.shape == (2, 4, 0, 64) and torch.autograd.grad(o.sum(), z)[0].shape == z.shape
    e = torch.zeros(0, 4, 64, device=DEV)
    c = torch.zeros(0, 2, 5, 64, device=DEV)
    assert la.causal_attention_step(e, e[:, :2], e[:, :2], c, c.clone(), torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 4, 64)


def test_refusals():
    q, k, v, _ = _inputs(2, 4, 2, 8, 64, "f32")
    for bad in (lambda: la.causal_attention(q, k[:, :, :4], v), lambda: la.causal_attention(q[:, :3], k, v), lambda: la.causal_attention(q.half(), k.half(), v.half()),
                lambda: la.causal_attention(q, k.bfloat16(), v), lambda: la.causal_attention(q[0], k[0], v[0]), lambda: la.causal_attention(q, k, v, cu_seqlens=[0, 8]),
                lambda: la.causal_attention(q, k, v.cpu()), lambda: la.causal_attention(*(torch.zeros(1, 1, 2, 136, device=DEV),) * 3)):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: la.causal_attention(q, k, v, float("inf")), lambda: la.causal_attention(q[:1], k[:1], v[:1], cu_seqlens=[0, 7])):
        with pytest.raises(ValueError):
            bad()
    q, k, v, kc, vc = _step_inputs(2, 4, 2, 9, 64, "f32")
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: la.causal_attention_step(q, k, v, kc, vc[:, :, :5], n), lambda: la.causal_attention_step(q, k, v, kc, vc, n.long()),
                lambda: la.causal_attention_step(q, k, v, kc[:, :1].expand(-1, 2, -1, -1), vc, n), lambda: la.causal_attention_step(q, k, v, kc.bfloat16(), vc, n),
                lambda: la.causal_attention_step(q, k, v, kc, vc, n[:1]), lambda: la.causal_attention_step(q.requires_grad_(), k, v, kc, vc, n)):
        with pytest.raises(RuntimeError):
            bad()
