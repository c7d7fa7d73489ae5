"""decay_linear_attention against its definition in float64, with elementwise bounds.

Bounds.  u' = 2^-23 (two units of float32 per addition), r = 2^-15 where operands enter products in two bfloat16 parts (each off by 2^-17 of itself, at
most three in a term) and 0 in float32.  Every result is a sum of terms, each a product with a decay: the bound is the sum of the terms' magnitudes times
  E = r + (T + dk + dv + 64) u' + (1 + |G|) 2^-20
-- one term passes at most T + dk + dv additions; the exponents' sums and the factors of the chunks between are good to a few units each, and |G| <= 16
stands for what the largest |sum of g| that leaves anything adds (x e^-x < 1 beyond) -- and eps / 2 of the value for the result's type.  dg is formed from sums of
x_s . out_s over the whole sequence where they go through the state, and over a chunk where they are pairs of it: those magnitudes, times 2 E (two dots)."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = {torch.bfloat16: 64, torch.float32: 32}


def _suffix(x):
    return x.flip(0).cumsum(0).flip(0)


def _formulas(q, k, v, g, s0, scale, do, ds, chunk):
    """One sequence and head in float64: results; with absolute inputs, their terms' magnitudes.  dg comes apart: its value, and the sums it is formed from."""
    T = q.shape[0]
    G = g.cumsum(0)
    keep = torch.ones(T, T, dtype=torch.bool, device=q.device).tril()
    E = torch.exp((G[:, None] - G[None, :]).masked_fill(~keep, -np.inf))
    into, last = torch.exp(G)[:, None], (torch.exp(G[-1:] - G)[:, None] if T else G[:, None])
    whole = torch.exp(G[-1]) if T else torch.ones((), dtype=q.dtype, device=q.device)
    P = scale * (q @ k.T) * E
    out = {"o": P @ v + scale * into * (q @ s0), "state": whole * s0 + (k * last).T @ v}
    if do is None:
        return out
    dP = scale * (do @ v.T) * E
    dqs, dks = scale * into * (do @ s0.T), last * (v @ ds.T)
    out.update(dq=dP @ k + dqs, dk=dP.T @ q + dks, dv=P.T @ do + last * (k @ ds), dstate=whole * ds + scale * (q * into).T @ do)
    A = P * (do @ v.T)
    before = A.cumsum(1) - A  # sum over r < t
    at = torch.arange(T, device=q.device)
    near = at[:, None] // chunk == at[None, :] // chunk
    out["dg"] = (before * keep).sum(0) + _suffix((dqs * q).sum(1)) + ((dks * k).sum(1).cumsum(0) - (dks * k).sum(1)) + whole * (ds * s0).sum()
    pairs, far = A * near, A * ~near
    in_chunk = torch.zeros(T, dtype=q.dtype, device=q.device)
    for c in range(0, T, chunk):
        in_chunk[c : c + chunk] = 2 * pairs[c : c + chunk].sum()
    out["dg sums"] = in_chunk + 2 * far.sum() + (dqs * q).sum() + (dks * k).sum() + (ds * out["state"]).sum()
    return out


def _close(got, ref, bound, what):
    eps = torch.finfo(got.dtype).eps / 2
    tol = bound * (1 + eps) + eps * ref.abs() + 1e-36
    worst = ((got.double() - ref).abs() / tol).nan_to_num(np.inf)
    assert got.shape == ref.shape and (worst.numel() == 0 or float(worst.max()) <= 1), f"{what}: {float(worst.max()):.2f} of the bound at {np.unravel_index(int(worst.argmax()), worst.shape)}"


def _inputs(B, H, T, dk, dv, dtype, *, rows=None, state=True, token_first=False, per_head=False, decay=0.3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: torch.randn(*s, generator=gen) * std

    def heads(d):
        t = n(B, T, H, d).to(DEV, DT[dtype]).transpose(1, 2)
        return t if token_first else t.contiguous()

    q, k, v, do = heads(dk), heads(dk), heads(dv), heads(dv)
    g = -decay * torch.rand(H, generator=gen) if per_head else -decay * torch.rand(B, H, T, generator=gen) * torch.exp(n(1, H, 1))
    rows = B if rows is None else rows
    return dict(q=q, k=k, v=v, g=g.to(DEV), s0=n(rows, H, dk, dv).to(DEV) if state else None), do, n(rows, H, dk, dv, std=0.3).to(DEV)


def _check(t, do, ds, *, scale=None, lens=None, cu=None):
    q, k, v, g, s0 = (t[x] for x in ("q", "k", "v", "g", "s0"))
    B, H, T, dk = q.shape
    dv, dt = v.shape[-1], q.dtype
    leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, v, g, s0)]
    if lens is not None and cu is None:
        cu = [0, *np.cumsum(lens).tolist()]
    o, sT = la.decay_linear_attention(*leaves[:4], scale, leaves[4], cu_seqlens=cu)
    with torch.no_grad():
        o2, sT2 = la.decay_linear_attention(q, k, v, g, scale, s0, cu_seqlens=cu)
    assert torch.equal(o, o2) and torch.equal(sT, sT2) and o.dtype == dt and sT.dtype == torch.float32
    wanted = [x for x in leaves if x is not None]
    grads = dict(zip([n for n, x in zip(("dq", "dk", "dv", "dg", "dstate"), leaves) if x is not None], torch.autograd.grad([o, sT], wanted, [do, ds])))
    for x, gr in zip(wanted, grads.values()):
        assert gr.shape == x.shape and gr.dtype == x.dtype
    sc = dk ** -0.5 if scale is None else scale
    E = (2.0 ** -15 if dt == torch.bfloat16 else 0.0) + (T + dk + dv + 64) * 2.0 ** -23 + 17 * 2.0 ** -20
    spans = [(b, 0, T, b) for b in range(B)] if lens is None else [(0, int(sum(lens[:i])), int(sum(lens[: i + 1])), i) for i in range(len(lens))]
    dgh = [torch.zeros(H, dtype=torch.float64, device=DEV) for _ in range(2)]
    for b, lo, hi, row in spans:
        for h in range(H):
            x = [y[b, h, lo:hi].double() for y in (q, k, v)]
            gg = (g[h].expand(hi - lo) if g.dim() == 1 else g[b, h, lo:hi]).double()
            st = torch.zeros(dk, dv, dtype=torch.float64, device=DEV) if s0 is None else s0[row, h].double()
            back = (do[b, h, lo:hi].double(), ds[row, h].double())
            ref = _formulas(*x, gg, st, sc, *back, CHUNK[dt])
            mag = _formulas(*(y.abs() for y in x), gg, st.abs(), abs(sc), *(y.abs() for y in back), CHUNK[dt])
            got = {"o": o[b, h, lo:hi].detach(), "state": sT[row, h].detach(), **{n: grads[n][b, h, lo:hi] for n in ("dq", "dk", "dv")}}
            if s0 is not None:
                got["dstate"] = grads["dstate"][row, h]
            for name, y in got.items():
                _close(y, ref[name], E * mag[name], f"{name} row {row} head {h}")
            if g.dim() == 1:
                dgh[0][h] += ref["dg"].sum()
                dgh[1][h] += (2 * E * mag["dg sums"]).sum() + (hi - lo + 16) * 2.0 ** -23 * ref["dg"].abs().sum()
            else:
                _close(grads["dg"][b, h, lo:hi], ref["dg"], 2 * E * mag["dg sums"], f"dg row {row} head {h}")
    if g.dim() == 1:
        _close(grads["dg"], dgh[0], dgh[1], "dg")
    return o, sT, grads


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 2, 15, 31, 32, 33, 48, 63, 64, 65, 100, 128, 200])
def test_lengths(T, dtype):
    _check(*_inputs(2, 2, T, 64, 64, dtype, token_first=T % 2 == 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(8, 8), (128, 128), (40, 72), (80, 96), (128, 64), (64, 256), (256, 128), (256, 256), (20, 12), (3, 5), (1, 1), (65, 130)])
def test_heads(dk, dv, dtype):
    _check(*_inputs(1, 2, 150, dk, dv, dtype, token_first=dk % 16 == 0, state=dk != 80))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("decay", [0.0, 0.01, 3.0, 10.0, 60.0])
def test_decays(decay, dtype):
    """From none to ones that leave nothing of the token before."""
    _check(*_inputs(2, 2, 140, 64, 64, dtype, decay=decay, seed=1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,T,dk,dv,token_first", [(2, 3, 130, 64, 64, True), (1, 2, 77, 40, 24, False), (1, 1, 1300, 64, 64, True)])
def test_one_decay_for_each_head(B, H, T, dk, dv, token_first, dtype):
    _check(*_inputs(B, H, T, dk, dv, dtype, per_head=True, token_first=token_first, seed=2))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,T,dk,dv,state", [(1, 1100, 64, 64, True), (2, 2051, 128, 64, False), (3, 1536, 64, 128, True), (1, 1030, 256, 40, True)])
def test_few_rows_in_segments(H, T, dk, dv, state, dtype):
    _check(*_inputs(1, H, T, dk, dv, dtype, state=state, token_first=True, decay=0.02, seed=3))


PACKED = [[5], [1, 1, 1], [64, 64], [0, 70, 0, 1, 130, 0], [63, 1, 65, 2, 31, 33, 32], [600, 0, 513, 512, 1, 511, 2], [1500, 40]]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("lens", PACKED, ids=lambda x: "-".join(map(str, x)))
def test_packed(lens, state, dtype):
    _check(*_inputs(1, 2, sum(lens), 64, 64, dtype, rows=len(lens), state=state, token_first=state, seed=4), lens=lens)


def test_packed_table_on_the_gpu_and_many_rows():
    lens = [3] * 300 + [200]
    t, do, ds = _inputs(1, 1, sum(lens), 64, 64, "bf16", rows=len(lens), seed=5)
    _check(t, do, ds, lens=lens, cu=torch.tensor([0, *np.cumsum(lens).tolist()], device=DEV))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
def test_scales(scale, dtype):
    _check(*_inputs(1, 2, 100, 64, 64, dtype, seed=6), scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_document_is_what_it_is_alone(dtype):
    """Bit for bit, whatever it is packed with -- neighbours that are not finite included."""
    lens = [70, 129, 40]
    t, do, ds = _inputs(1, 2, sum(lens), 64, 64, dtype, rows=3, seed=7)
    for x in (t["q"], t["k"], t["v"], do):
        x[:, :, :70] = float("nan")
        x[:, :, 199:] = float("inf")
    leaves = {n: x.detach().requires_grad_() for n, x in t.items()}
    o, sT = la.decay_linear_attention(leaves["q"], leaves["k"], leaves["v"], leaves["g"], None, leaves["s0"], cu_seqlens=[0, 70, 199, 239])
    grads = torch.autograd.grad([o, sT], list(leaves.values()), [do, ds])
    one = {n: (x[1:2] if n == "s0" else x[:, :, 70:199]).detach().requires_grad_() for n, x in t.items()}
    o1, s1 = la.decay_linear_attention(one["q"], one["k"], one["v"], one["g"], None, one["s0"])
    want = torch.autograd.grad([o1, s1], list(one.values()), [do[:, :, 70:199], ds[1:2]])
    assert torch.equal(o[:, :, 70:199], o1) and torch.equal(sT[1:2], s1) and bool(torch.isfinite(o1).all())
    for a, b, n in zip(grads, want, t):
        assert torch.equal(a[1:2] if n == "s0" else a[:, :, 70:199], b) and bool(torch.isfinite(b).all()), n


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_reset_drops_what_came_before(dtype):
    """g = -inf at a token: from there on as if the sequence began."""
    t, do, ds = _inputs(1, 2, 150, 64, 64, dtype, seed=8)
    for at in (0, 40, 64, 100):
        g = t["g"].clone()
        g[:, :, at] = -float("inf")
        o, sT = la.decay_linear_attention(t["q"], t["k"], t["v"], g, None, t["s0"])
        cut = [t[n][:, :, at:] for n in ("q", "k", "v", "g")]
        o1, s1 = la.decay_linear_attention(*cut)
        big = float(o1.float().abs().max())
        assert torch.allclose(o[:, :, at:].float(), o1.float(), rtol=2 * torch.finfo(o.dtype).eps, atol=1e-5 * big) and torch.allclose(sT, s1, rtol=1e-5, atol=1e-4)
        if at:
            o2, _ = la.decay_linear_attention(*(t[n][:, :, :at] for n in ("q", "k", "v", "g")), None, t["s0"])
            assert torch.allclose(o[:, :, :at].float(), o2.float(), rtol=2 * torch.finfo(o.dtype).eps, atol=1e-5 * big)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_values_that_are_not_finite_stay_behind_their_token(which, value, dtype):
    """Outputs of earlier tokens of the same chunk, and of other heads, are what they are without them; from the token on they are not finite."""
    t, do, ds = _inputs(1, 2, 100, 64, 64, dtype, seed=9)
    o, _ = la.decay_linear_attention(t["q"], t["k"], t["v"], t["g"], None, t["s0"])
    bad = {**t, which: t[which].clone()}
    bad[which][0, 1, 70, 5] = value
    o2, s2 = la.decay_linear_attention(bad["q"], bad["k"], bad["v"], bad["g"], None, bad["s0"])
    assert torch.equal(o2[:, 0], o[:, 0]) and torch.equal(o2[:, 1, :70], o[:, 1, :70])
    if which == "q":
        assert not bool(torch.isfinite(o2[0, 1, 70]).any()) and torch.equal(o2[:, 1, 71:], o[:, 1, 71:]) and bool(torch.isfinite(s2).all())
    elif which == "k":
        assert not bool(torch.isfinite(o2[0, 1, 70:]).any()) and not bool(torch.isfinite(s2[0, 1, 5]).any()) and bool(torch.isfinite(s2[0, 0]).all())
    else:  # one column of the values
        rest = torch.arange(64, device=DEV) != 5
        assert not bool(torch.isfinite(o2[0, 1, 70:, 5]).any()) and torch.equal(o2[0, 1, :, rest], o[0, 1, :, rest])
        assert not bool(torch.isfinite(s2[0, 1, :, 5]).any()) and bool(torch.isfinite(s2[0, 1][:, rest]).all())


def test_gradients_of_values_that_are_not_finite_stay_before_their_token():
    t, do, ds = _inputs(1, 1, 100, 64, 64, "bf16", seed=10)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o, sT = la.decay_linear_attention(*leaves, t["g"])
    want = torch.autograd.grad(o, leaves, do, retain_graph=True)
    bad = do.clone()
    bad[0, 0, 30, 7] = float("inf")
    got = torch.autograd.grad(o, leaves, bad)
    keep = torch.arange(100, device=DEV) > 30
    assert torch.equal(got[0][:, :, keep], want[0][:, :, keep]) and torch.equal(got[1][:, :, keep], want[1][:, :, keep]) and torch.equal(got[2][:, :, keep], want[2][:, :, keep])
    assert torch.equal(got[0][:, :, :30], want[0][:, :, :30]) and not bool(torch.isfinite(got[2][0, 0, :31, 7]).any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_and_memory_orders(dtype):
    t, do, ds = _inputs(2, 3, 90, 64, 32, dtype, seed=11)
    o, sT = la.decay_linear_attention(t["q"], t["k"], t["v"], t["g"], None, t["s0"])
    wide = torch.cat([t[n].transpose(1, 2).reshape(2, 90, -1) for n in ("q", "k", "v")], 2)  # one projection
    q, k = (wide[:, :, i * 192 : (i + 1) * 192].view(2, 90, 3, 64).transpose(1, 2) for i in range(2))
    v = wide[:, :, 384:].view(2, 90, 3, 32).transpose(1, 2)
    g = t["g"].transpose(1, 2).contiguous().transpose(1, 2)
    o2, s2 = la.decay_linear_attention(q, k, v, g, None, t["s0"].transpose(2, 3).contiguous().transpose(2, 3))
    assert torch.equal(o, o2) and torch.equal(sT, s2) and o2.stride(1) < o2.stride(2)
    shared = t["k"][:, :1].expand(-1, 3, -1, -1)  # one key head for all
    o3, _ = la.decay_linear_attention(t["q"], shared, t["v"], t["g"])
    o4, _ = la.decay_linear_attention(t["q"], shared.contiguous(), t["v"], t["g"])
    assert torch.equal(o3, o4)
    off = torch.empty(t["q"].numel() + 1, device=DEV, dtype=DT[dtype])[1:].view(t["q"].shape).copy_(t["q"])  # rows that start beside a 16-byte boundary
    assert torch.equal(la.decay_linear_attention(off, t["k"], t["v"], t["g"], None, t["s0"])[0], o)
    leaf = t["k"][:, :1].clone().requires_grad_()
    o5, _ = la.decay_linear_attention(t["q"], leaf.expand(-1, 3, -1, -1), t["v"], t["g"])
    full = shared.contiguous().requires_grad_()
    o6, _ = la.decay_linear_attention(t["q"], full, t["v"], t["g"])
    a, b = torch.autograd.grad(o5, leaf, do)[0], torch.autograd.grad(o6, full, do)[0].float().sum(1, True)
    assert torch.allclose(a.float(), b, rtol=4 * torch.finfo(a.dtype).eps, atol=4 * torch.finfo(a.dtype).eps * float(b.abs().max()))
    one = torch.autograd.grad(la.decay_linear_attention(full, full, t["v"], t["g"])[0].sum(), full)[0]  # a broadcast gradient, one tensor twice
    two = [x.detach().requires_grad_() for x in (full, full)]
    x, y = torch.autograd.grad(la.decay_linear_attention(*two, t["v"], t["g"])[0], two, torch.ones_like(do))
    assert torch.equal(one, x + y)


def test_types_of_gates_and_states():
    t, do, ds = _inputs(1, 2, 40, 64, 64, "bf16", seed=12)
    half = {n: t[n].bfloat16() for n in ("g", "s0")}
    leaves = [half[n].detach().requires_grad_() for n in ("g", "s0")]
    o, sT = la.decay_linear_attention(t["q"], t["k"], t["v"], leaves[0], None, leaves[1])
    o2, s2 = la.decay_linear_attention(t["q"], t["k"], t["v"], half["g"].float(), None, half["s0"].float())
    assert torch.equal(o, o2) and torch.equal(sT, s2)
    assert [x.dtype for x in torch.autograd.grad([o, sT], leaves, [do, ds])] == [torch.bfloat16] * 2


def test_one_output_alone():
    t, do, ds = _inputs(1, 2, 90, 64, 64, "f32", seed=13)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
    o, sT = la.decay_linear_attention(*leaves[:4], None, leaves[4])
    both = torch.autograd.grad([o, sT], leaves, [do, ds], retain_graph=True)
    by_o = torch.autograd.grad(o, leaves, do, retain_graph=True)
    by_s = torch.autograd.grad(sT, leaves, ds, allow_unused=True)
    for a, b, c in zip(both, by_o, by_s):
        assert torch.allclose(a, b + (0 if c is None else c), rtol=1e-4, atol=1e-4 * float(a.abs().max()))


def test_gradients_against_differences():
    """Central differences in float32 with steps of 1e-2: the remainder is step^2 of a third derivative of order one."""
    t, do, ds = _inputs(1, 2, 40, 16, 8, "f32", seed=14, decay=0.5)
    leaves = {n: x.detach().requires_grad_() for n, x in t.items()}

    def loss(a):
        o, sT = la.decay_linear_attention(a["q"], a["k"], a["v"], a["g"], None, a["s0"])
        return (o * do).double().sum() + (sT * ds).double().sum()

    grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    gen = torch.Generator().manual_seed(9)
    for n, x in t.items():
        dirn, step = torch.randn(x.shape, generator=gen).to(DEV), 1e-2
        diff = (loss({**t, n: x + step * dirn}) - loss({**t, n: x - step * dirn})) / (2 * step)
        assert abs(float(diff - (grads[n].double() * dirn).sum())) < 1e-2 * float((grads[n].double() * dirn).abs().sum()), n


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T", [200, 1100])
def test_repeats_bit_for_bit_and_replays(T, packed):
    lens = [T - 60, 0, 60]
    t, do, ds = _inputs(1, 2, T, 64, 64, "bf16", rows=3 if packed else None, seed=15)
    cu = torch.tensor([0, *np.cumsum(lens).tolist()], dtype=torch.int32, device=DEV) if packed else None
    leaves = [t[n].detach().clone().requires_grad_() for n in ("q", "k", "v", "g", "s0")]

    def both():
        o, sT = la.decay_linear_attention(*leaves[:4], None, leaves[4], cu_seqlens=cu)
        return (o, sT, *torch.autograd.grad([o, sT], leaves, [do, ds]))

    assert all(torch.equal(a, b) for a, b in zip(both(), both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(leaves[0]))
            if packed:
                cu[1:3] = T - 100 - i
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both()))


def test_refused_while_a_graph_of_the_leaf_is_alive():
    x = torch.randn(1, 2, 40, 64, device=DEV, requires_grad=True)
    g = -torch.ones(2, device=DEV)
    alive = la.decay_linear_attention(x, x, x, g)
    graph, keep = torch.cuda.CUDAGraph(), torch.zeros(8, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        keep.add_(1)
        with pytest.raises(RuntimeError, match="alive"):
            la.decay_linear_attention(x, x, x, g)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((keep == 1).all()) and bool(torch.isfinite(alive[0]).all())


def test_rows_beyond_two_to_the_31_elements():
    """Tokens 2^16 elements apart: 40000 of them reach behind 2^31."""
    T = 40000
    big = torch.zeros(T, 65536, dtype=torch.bfloat16, device=DEV)
    t, _, _ = _inputs(1, 2, T, 64, 64, "bf16", seed=16, state=False)
    views = []
    for i, n in enumerate(("q", "k", "v")):
        w = big[:, i * 128 : i * 128 + 128].view(T, 2, 64).transpose(0, 1)[None]
        w.copy_(t[n])
        views.append(w)
    o, sT = la.decay_linear_attention(*views, t["g"])
    o2, s2 = la.decay_linear_attention(t["q"], t["k"], t["v"], t["g"])
    assert torch.equal(o, o2) and torch.equal(sT, s2)


def test_empty():
    e = torch.zeros(0, 2, 5, 64, device=DEV, requires_grad=True)
    o, s = la.decay_linear_attention(e, e, e, torch.zeros(2, device=DEV))
    assert o.shape == (0, 2, 5, 64) and s.shape == (0, 2, 64, 64)
    z = torch.zeros(2, 2, 0, 64, device=DEV, requires_grad=True)
    s0 = torch.randn(2, 2, 64, 64, device=DEV, requires_grad=True)
    g = torch.zeros(2, device=DEV, requires_grad=True)
    o, s = la.decay_linear_attention(z, z, z, g, None, s0)
    assert o.shape == z.shape and torch.equal(s, s0)
    gz, gs, gg = torch.autograd.grad(s, [z, s0, g], torch.ones_like(s))
    assert gz.shape == z.shape and bool((gs == 1).all()) and bool((gg == 0).all())


# -- one token --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (3, 2, 64, 64), (2, 5, 128, 128), (2, 2, 80, 96), (1, 3, 256, 200), (2, 2, 33, 7), (1, 2, 64, 512), (40, 8, 128, 130)])
def test_step(B, H, dk, dv, inplace, dtype):
    """o and the state within the roundings of their sums: dk additions and one of the state."""
    t, _, _ = _inputs(B, H, 1, dk, dv, dtype, seed=17)
    q, k, v, g = (t[n][:, :, 0] for n in ("q", "k", "v", "g"))
    S = t["s0"].double() * torch.exp(g.double())[..., None, None] + k.double()[..., :, None] * v.double()[..., None, :]
    mag = t["s0"].double().abs() * torch.exp(g.double())[..., None, None] + (k.double()[..., :, None] * v.double()[..., None, :]).abs()
    want = (q.double()[..., None] * S).sum(-2) * dk ** -0.5
    wmag = (q.double().abs()[..., None] * mag).sum(-2) * dk ** -0.5
    state = t["s0"].clone()
    o, s1 = la.decay_linear_attention_step(q, k, v, g, state, inplace=inplace)
    assert (s1 is state) if inplace else torch.equal(state, t["s0"])
    _close(s1, S, 2.0 ** -20 * mag, "state")
    _close(o, want, (2.0 ** -20 + (dk + 16) * 2.0 ** -23) * wmag, "o")


def test_step_with_one_decay_for_each_head_and_gradients():
    t, _, _ = _inputs(2, 3, 1, 64, 32, "f32", per_head=True, seed=18)
    q, k, v = (t[n][:, :, 0] for n in ("q", "k", "v"))
    o, s = la.decay_linear_attention_step(q, k, v, t["g"], t["s0"])
    o2, s2 = la.decay_linear_attention_step(q, k, v, t["g"].expand(2, 3), t["s0"])
    assert torch.equal(o, o2) and torch.equal(s, s2)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, t["g"], t["s0"])]
    og, sg = la.decay_linear_attention_step(*leaves)
    assert torch.allclose(og, o, rtol=1e-4, atol=1e-4) and torch.allclose(sg, s, rtol=1e-4, atol=1e-4)
    assert all(bool(torch.isfinite(x).all()) and x.shape == y.shape for x, y in zip(torch.autograd.grad([og.sum(), sg.sum()], leaves), leaves))
    with pytest.raises(RuntimeError, match="in place"):
        la.decay_linear_attention_step(*leaves, inplace=True)


def test_prompt_then_tokens_in_a_replayed_graph():
    t, _, _ = _inputs(2, 2, 80, 64, 64, "f32", seed=19)
    whole, last = la.decay_linear_attention(t["q"], t["k"], t["v"], t["g"], None, t["s0"])
    _, state = la.decay_linear_attention(*(t[n][:, :, :70] for n in ("q", "k", "v", "g")), None, t["s0"])
    tok = [t[n][:, :, 70].clone() for n in ("q", "k", "v", "g")]
    graph, keep = torch.cuda.CUDAGraph(), state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        la.decay_linear_attention_step(*tok, keep, inplace=True)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        o, _ = la.decay_linear_attention_step(*tok, state, inplace=True)
    for i in range(70, 80):
        for buf, n in zip(tok, ("q", "k", "v", "g")):
            buf.copy_(t[n][:, :, i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(o, whole[:, :, i], rtol=1e-4, atol=1e-4)
    assert torch.allclose(state, last, rtol=1e-4, atol=1e-4)


def test_step_counts_as_a_write():
    t, _, _ = _inputs(1, 2, 1, 64, 64, "f32")
    state = t["s0"].clone()
    out = (torch.ones(1, device=DEV, requires_grad=True) * state).sum()
    la.decay_linear_attention_step(*(t[n][:, :, 0] for n in ("q", "k", "v", "g")), state, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_refusals():
    t, _, _ = _inputs(2, 2, 8, 64, 64, "f32")
    q, k, v, g, s = (t[n] for n in ("q", "k", "v", "g", "s0"))
    f = la.decay_linear_attention
    wide = torch.zeros(1, 1, 2, 264, device=DEV)
    for bad in (lambda: f(q, k[:, :, :4], v, g), lambda: f(q, k, v[:, :1], g), lambda: f(q.half(), k.half(), v.half(), g), lambda: f(q, k.bfloat16(), v, g), lambda: f(q[0], k[0], v[0], g[0]),
                lambda: f(q, k, v, g[:, :, :3]), lambda: f(q, k, v, g[0, 0]), lambda: f(q, k, v, g.int()), lambda: f(q, k, v, g, None, s[:1]), lambda: f(q, k, v, g, None, s[..., :8]),
                lambda: f(q, k, v, g.cpu()), lambda: f(q.cpu(), k, v, g), lambda: f(q, k, v, g, cu_seqlens=[0, 8]), lambda: f(wide, wide, wide, torch.zeros(1, device=DEV)),
                lambda: la.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], s.bfloat16(), inplace=True),
                lambda: la.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], s[:1]), lambda: la.decay_linear_attention_step(q, k, v, g, s)):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: f(q, k, v, g, float("nan")), lambda: f(q[:1], k[:1], v[:1], g[:1], cu_seqlens=[0, 7])):
        with pytest.raises(ValueError):
            bad()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            f(torch.autograd.forward_ad.make_dual(q, q), k, v, g)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("T", [40, 600])
def test_states_and_gates_gradients_of_bf16_are_as_exact_as_fp32(T, per_head):
    """By norms.  A state is T / 64 chunks, each a scaling and six products into one sum: 7 T / 64 roundings of 2^-24, in no step with each other, and factors
    good to three units of 2^-23: 3 2^-23 + (7 T / 64)^(1/2) 2^-24 < 2^-20.  dg is made of two such states' dots, whose own sums are as long: 2^-19.  Operands in two parts
    would leave 2^-18 and 2^-17."""
    t, do, ds = _inputs(2, 3, T, 128, 128, "bf16", per_head=per_head, decay=0.02, seed=31)
    leaves = {n: x.detach().requires_grad_() for n, x in t.items()}
    o, sT = la.decay_linear_attention(leaves["q"], leaves["k"], leaves["v"], leaves["g"], None, leaves["s0"])
    dg, d0 = torch.autograd.grad([o, sT], [leaves["g"], leaves["s0"]], [do, ds])
    want = {"state": torch.empty_like(sT, dtype=torch.float64), "dstate": torch.empty_like(sT, dtype=torch.float64), "dg": torch.zeros_like(dg, dtype=torch.float64)}
    for b in range(2):
        for h in range(3):
            g = t["g"][h].expand(T) if per_head else t["g"][b, h]
            r = _formulas(*(t[n][b, h].double() for n in ("q", "k", "v")), g.double(), t["s0"][b, h].double(), 128 ** -0.5, do[b, h].double(), ds[b, h].double(), 64)
            want["state"][b, h], want["dstate"][b, h] = r["state"], r["dstate"]
            if per_head:
                want["dg"][h] += r["dg"].sum()
            else:
                want["dg"][b, h] = r["dg"]
    for what, got, tol in (("state", sT, 2.0 ** -20), ("dstate", d0, 2.0 ** -20), ("dg", dg, 2.0 ** -19)):
        off = float((got.detach().double() - want[what]).norm() / want[what].norm())
        assert off < tol, f"{what}: {off:.2g}"


@pytest.mark.parametrize("T", [100, 700])
def test_gates_gradient_does_not_depend_on_who_wants_the_states(T):
    t, do, ds = _inputs(1, 2, T, 64, 64, "bf16", seed=32)
    grads = []
    for wanted in (True, False):
        g, s0 = t["g"].detach().requires_grad_(), t["s0"].detach().requires_grad_(wanted)
        o, sT = la.decay_linear_attention(t["q"], t["k"], t["v"], g, None, s0)
        grads.append(torch.autograd.grad([o, sT], [g, s0] if wanted else [g], [do, ds])[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,T,dv", [(130, 9001, 8), (64, 17100, 40), (3, 8193, 256)])
def test_gates_gradients_over_segments_of_more_than_4096_tokens(H, T, dv, dtype):
    """By norms, as above: at most nine roundings a chunk of 32, 3 2^-23 + (9 T / 32)^(1/2) 2^-24 < 2^-17 of a state, twice that of dg.  The definition token by token."""
    t, do, ds = _inputs(1, H, T, 8, dv, dtype, state=False, decay=0.02, seed=33)
    g = t["g"].detach().requires_grad_()
    o, sT = la.decay_linear_attention(t["q"], t["k"], t["v"], g)
    got = torch.autograd.grad([o, sT], [g], [do, ds])[0]
    q, k, v, d = (x[0].transpose(0, 1).double() for x in (t["q"], t["k"], t["v"], do))  # [T, H, .]
    e = torch.exp(t["g"][0].double()).T[:, :, None, None]
    kv, qd = k[..., :, None] * v[..., None, :], 8 ** -0.5 * q[..., :, None] * d[..., None, :]
    before, s = torch.empty_like(kv), torch.zeros_like(kv[0])
    for i in range(T):
        before[i] = s
        s = e[i] * s + kv[i]
    want, back = torch.empty(T, H, dtype=torch.float64, device=DEV), ds[0].double()
    for i in range(T - 1, -1, -1):
        back = back + qd[i]  # of the state behind token i
        want[i] = (e[i] * back * before[i]).sum((1, 2))
        back = e[i] * back
    off = float((got[0].T.double() - want).norm() / want.norm())
    assert off < 2.0 ** -16, f"{off:.2g}"
