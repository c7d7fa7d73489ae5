"""The gated linear recurrence against its definition, token by token in float64, with elementwise bounds.

Bounds.  With u = 2^-24 and M_t = a_t M_{t-1} + |x_t| (the recurrence on magnitudes) one step h = e^g h + x in float32 adds at
most u (4 + 2 |g_t|) M_t: e^g comes from a product with log2(e), whose rounding moves the result by |g| u, twice for the rounding of
the constant, and an exponential good to one unit in the last place (2 u), then a product and a sum (u each).  Errors travel with
the recurrence itself: E_t = a_t E_{t-1} + u (4 + 2 |g_t|) M_t.  Joining spans in a tree instead of one by one adds a product and a
sum per level, at most as many again: 2 E_t.  An output of type t is rounded once: eps_t / 2 |h|.  The gradients are the same
recurrence backwards; dg = h_{t-1} o_t with o_t = a_t dh_t adds its factors' errors and one rounding."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TINY = 1e-36  # results that leave float32's normal range
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _scan(x, g, h0):
    """h, its bound, the magnitudes, row by row of [T, D] float64 arrays; h0 exact."""
    h, E, M = h0.copy(), np.zeros_like(h0), np.abs(h0)
    H, EE = np.empty_like(x), np.empty_like(x)
    a = np.exp(g)
    for t in range(x.shape[0]):
        M = a[t] * M + np.abs(x[t])
        h = a[t] * h + x[t]
        E = a[t] * E + U * (4 + 2 * np.abs(np.maximum(g[t], -200))) * M
        H[t], EE[t] = h, 2 * E
    return H, EE


def _reference(x, g, h0, dy, ds):
    H, E = _scan(x, g, h0)
    T = x.shape[0]
    a = np.exp(g)
    ga = np.abs(np.maximum(g, -200))
    o, Eo, M = ds.copy(), np.zeros_like(ds), np.abs(ds)
    dx, dg, Edx, Edg = (np.empty_like(x) for _ in range(4))
    for t in range(T - 1, -1, -1):
        dh, Edh, M = dy[t] + o, Eo, M + np.abs(dy[t])
        dx[t], Edx[t] = dh, 2 * Edh + U * M
        o, Eo, M = a[t] * dh, a[t] * Edh + U * (4 + 2 * ga[t]) * a[t] * M, a[t] * M
        before, Eb = (H[t - 1], E[t - 1]) if t else (h0, np.zeros_like(h0))
        dg[t] = before * o
        Edg[t] = np.abs(before) * 2 * Eo + np.abs(o) * Eb + 2 * U * np.abs(dg[t])
    return H, E, dx, Edx, dg, Edg, o, 2 * Eo


def _np(t):
    return t.detach().double().cpu().numpy()


def _within(got, ref, bound, what):
    eps = torch.finfo(got.dtype).eps / 2
    got = _np(got)
    tol = bound * (1 + 2 * eps) + eps * np.abs(ref) + TINY
    off = np.abs(got - ref) - tol
    assert np.all(off <= 0), f"{what}: off by {np.max(np.abs(got - ref) / tol):.2f} of the bound at {np.unravel_index(np.argmax(off), off.shape)}"


def _inputs(B, T, D, dtype, g_dtype, rows, seed=0, strided=False):
    r = torch.Generator().manual_seed(seed)
    wide = torch.randn(B, T, 2 * D + 16, generator=r)
    x = wide[..., :D] if strided else wide[..., :D].contiguous()
    rate = torch.exp(-torch.rand(D, generator=r) * 6)
    g = -rate * torch.nn.functional.softplus(torch.randn(B, T, D, generator=r))
    x = x.to(DEV, DT[dtype]) if not strided else wide.to(DEV, DT[dtype])[..., 8 : 8 + D]
    g = g.to(DEV, DT[g_dtype])
    if strided:
        both = torch.empty(B, T, D + 8, device=DEV, dtype=g.dtype)
        both[..., :D] = g
        g = both[..., :D]
    s0 = torch.randn(rows, D, generator=r).to(DEV)
    dy = torch.randn(B, T, D, generator=r).to(DEV, DT[dtype])
    ds = torch.randn(rows, D, generator=r).to(DEV)
    return x, g, s0, dy, ds


def _check(x, g, s0, dy, ds, cu=None, state=True):
    leaves = [x.detach().requires_grad_(), g.detach().requires_grad_()] + ([s0.detach().requires_grad_()] if state else [])
    y, sT = la.gated_linear_recurrence(*leaves, cu_seqlens=cu)
    assert y.dtype == x.dtype and y.shape == x.shape and sT.dtype == torch.float32
    grads = torch.autograd.grad([y, sT], leaves, [dy, ds])
    with torch.no_grad():  # the call without gradients is the same function
        y2, sT2 = la.gated_linear_recurrence(x, g, s0 if state else None, cu_seqlens=cu)
    assert torch.equal(y, y2) and torch.equal(sT, sT2)
    rows = [(i, 0, x.shape[1]) for i in range(x.shape[0])] if cu is None else [(0, a, b) for a, b in zip(cu[:-1], cu[1:])]
    nx, ng, ns, ndy, nds = (_np(t) for t in (x, g, s0, dy, ds))
    for i, (b, lo, hi) in enumerate(rows):
        h0 = ns[i] if state else np.zeros_like(ns[i])
        H, E, dx, Edx, dg, Edg, d0, Ed0 = _reference(nx[b, lo:hi], ng[b, lo:hi], h0, ndy[b, lo:hi], nds[i])
        _within(y[b, lo:hi], H, E, "y")
        _within(sT[i], H[-1] if hi > lo else h0, E[-1] if hi > lo else 0 * h0, "final state")
        _within(grads[0][b, lo:hi], dx, Edx, "dx")
        _within(grads[1][b, lo:hi], dg, Edg, "dg")
        if state:
            _within(grads[2][i], d0, Ed0, "d_initial_state")


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 1, 64), (3, 2, 65), (2, 4, 8), (1, 127, 40), (2, 128, 64), (1, 129, 33), (2, 255, 24), (1, 256, 72),
                                   (2, 257, 130), (1, 1000, 66), (1, 3001, 64), (1, 5000, 20)])
def test_forward_and_gradients(B, T, D, types):
    _check(*_inputs(B, T, D, *types, rows=B), state=(T % 2 == 1))


def test_one_long_row():
    """More than 1024 tiles of 128 tokens of few channels: pairs of one tile, of 32 and published states all take part."""
    _check(*_inputs(1, 135_000, 3, "bf16", "f32", rows=1))


def test_chained_tiles_repeat_bit_for_bit():
    x, g, s0, dy, ds = _inputs(1, 20_000, 64, "bf16", "bf16", rows=1)
    leaves = [t.detach().requires_grad_() for t in (x, g, s0)]

    def both():
        y, sT = la.gated_linear_recurrence(*leaves)
        return (y, sT, *torch.autograd.grad([y, sT], leaves, [dy, ds]))

    first = both()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, both()))


def test_two_streams_at_once():
    """Calls that overlap on two streams have workspaces of their own."""
    sets = [_inputs(1, 9000, 256, "bf16", "f32", rows=1, seed=s)[:3] for s in (1, 2)]
    want = [la.gated_linear_recurrence(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(la.gated_linear_recurrence(*sets[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w[0], y) and torch.equal(w[1], s) for y, s in g)


@pytest.mark.parametrize("types", [("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [0, 5, 0, 0, 300, 1, 0], [128, 256, 127, 129], [2500, 3, 1024]], ids=str)
def test_packed(lens, types):
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    _check(*_inputs(1, cu[-1], 48, *types, rows=len(lens)), cu=cu)


@pytest.mark.parametrize("kind", ["uneven", "short", "long", "uneven more", "short more"])
def test_packed_rows_of_every_kind(kind):
    """More rows than a wave looks at in one go, with empty ones; one row of more than 1024 tiles behind short ones."""
    r = np.random.default_rng(3)
    lens = {"uneven": (r.integers(0, 5, 700) * (r.random(700) < 0.5)).tolist() + [2000, 0, 129, 0], "short": [1, 0, 2] * 1500, "long": [5, 0, 132_000, 0, 900]}
    lens |= {"uneven more": lens["uneven"] + [7000, 1, 0, 300], "short more": lens["short"] * 2}
    lens = lens[kind]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    _check(*_inputs(1, cu[-1], 3 if kind == "long" else 70, "bf16", "f32", rows=len(lens)), cu=cu)


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("D", [64, 51])
def test_strided_inputs(D, types):
    x, g, s0, dy, ds = _inputs(2, 300, D, *types, rows=2, strided=True)
    assert not x.is_contiguous() and not g.is_contiguous()
    _check(x, g, s0, dy, ds)
    _check(x.transpose(0, 1).contiguous().transpose(0, 1), g, s0, dy[:1].expand(2, -1, -1), ds)
    _check(x[::2].expand(2, -1, -1), g, s0, dy, ds)


def test_reset_gates():
    """-inf is a factor of 0: the row is two documents, and gradients stop there."""
    x, g, s0, dy, ds = _inputs(1, 700, 64, "f32", "f32", rows=1)
    g[:, 333] = -float("inf")
    leaves = [t.detach().requires_grad_() for t in (x, g, s0)]
    y, sT = la.gated_linear_recurrence(*leaves)
    grads = torch.autograd.grad([y, sT], leaves, [dy, ds])
    first, mid = la.gated_linear_recurrence(x[:, :333], g[:, :333], s0)
    g2 = g[:, 333:].clone()
    g2[:, 0] = 0
    second, last = la.gated_linear_recurrence(x[:, 333:], g2)
    assert torch.allclose(y, torch.cat([first, second], 1), rtol=1e-5, atol=1e-5) and torch.allclose(sT, last, rtol=1e-5, atol=1e-5)
    assert all(bool(torch.isfinite(t).all()) for t in grads) and bool((grads[1][:, 333] == 0).all())


def test_values_that_are_not_finite_stay_where_they_belong():
    """A NaN reaches its own channel from its own token on, nothing else; in the gradients its own sequence's channel alone."""
    x, g, s0, dy, ds = _inputs(1, 900, 24, "bf16", "f32", rows=2)
    cu = [0, 400, 900]
    clean = la.gated_linear_recurrence(x, g, s0, cu_seqlens=cu)
    x[0, 150, 5] = float("nan")
    leaves = [t.detach().requires_grad_() for t in (x, g, s0)]
    y, sT = la.gated_linear_recurrence(*leaves, cu_seqlens=cu)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 150:400, 5] = True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], clean[0][~bad])
    assert torch.isnan(sT).sum() == 1 and bool(torch.isnan(sT[0, 5]))
    dx, dg, d0 = torch.autograd.grad([y, sT], leaves, [dy, ds])
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(d0).all())
    assert bool(torch.isnan(dg[0, 151:400, 5]).all()) and torch.isnan(dg).sum() == 249


def test_one_gradient_alone():
    x, g, s0, dy, ds = _inputs(2, 300, 64, "f32", "f32", rows=2)
    leaves = [t.detach().requires_grad_() for t in (x, g, s0)]
    y, sT = la.gated_linear_recurrence(*leaves)
    both = torch.autograd.grad([y, sT], leaves, [dy, ds], retain_graph=True)
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    only_s = torch.autograd.grad(sT, leaves, ds)
    for a, b, c in zip(both, only_y, only_s):
        assert torch.allclose(a, b + c, rtol=1e-4, atol=1e-4)


def test_gradients_against_differences():
    """Central differences of the op itself in float32: the loss is linear in x and s0, so the step can be large; the second-order
    remainder in g is bounded by step^2 times the third derivative, below 1e-3 of the gradient here."""
    x, g, s0, dy, ds = _inputs(1, 40, 4, "f32", "f32", rows=1, seed=3)
    leaves = [t.detach().requires_grad_() for t in (x, g, s0)]

    def loss(*t):
        y, sT = la.gated_linear_recurrence(*t)
        return ((y * dy).double().sum() + (sT * ds).double().sum())

    grads = torch.autograd.grad(loss(*leaves), leaves)
    r = torch.Generator().manual_seed(5)
    for i, step in enumerate((1.0, 2e-2, 1.0)):
        v = torch.randn(leaves[i].shape, generator=r).to(DEV)
        args = [t.detach() for t in leaves]
        args[i] = leaves[i].detach() + step * v
        up = loss(*args)
        args[i] = leaves[i].detach() - step * v
        diff = (up - loss(*args)) / (2 * step)
        want = (grads[i].double() * v).sum()
        scale = (grads[i].double().abs() * v.abs()).sum()
        assert abs(float(diff - want)) < 1e-3 * float(scale)


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("B,D", [(1, 1), (3, 66), (2, 4096), (27, 1000), (5, 7)])
def test_step_is_one_token(B, D, types):
    x, g, s0, _, _ = _inputs(B, 1, D, *types, rows=B)
    y, sT = la.gated_linear_recurrence_step(x[:, 0], g[:, 0], s0)
    a, h0, nx = np.exp(_np(g[:, 0])), _np(s0), _np(x[:, 0])
    ref = a * h0 + nx
    bound = U * (4 + 2 * np.abs(_np(g[:, 0]))) * (np.abs(a * h0) + np.abs(nx))
    _within(sT, ref, bound, "state")
    _within(y, ref, bound, "y")
    again = s0.clone()
    y2, same = la.gated_linear_recurrence_step(x[:, 0], g[:, 0], again, inplace=True)
    assert same is again and torch.equal(again, sT) and torch.equal(y2, y)
    leaves = [t.detach().requires_grad_() for t in (x[:, 0], g[:, 0], s0)]
    with pytest.raises(RuntimeError, match="in place"):
        la.gated_linear_recurrence_step(*leaves, inplace=True)
    yg, sg = la.gated_linear_recurrence_step(*leaves)
    grads = torch.autograd.grad(sg, leaves, torch.ones_like(sg))
    assert torch.allclose(grads[2], torch.exp(g[:, 0].float()), rtol=1e-5)


def test_prompt_then_tokens_is_the_whole_sequence():
    x, g, s0, _, _ = _inputs(2, 300, 64, "f32", "f32", rows=2)
    y, sT = la.gated_linear_recurrence(x, g, s0)
    part, s = la.gated_linear_recurrence(x[:, :290], g[:, :290], s0)
    outs = [part]
    for t in range(290, 300):
        o, _ = la.gated_linear_recurrence_step(x[:, t], g[:, t], s, inplace=True)
        outs.append(o[:, None])
    assert torch.allclose(torch.cat(outs, 1), y, rtol=1e-5, atol=1e-5) and torch.allclose(s, sT, rtol=1e-5, atol=1e-5)


def test_captured_forward_and_backward_replay():
    x, g, s0, dy, ds = _inputs(1, 4100, 64, "bf16", "f32", rows=1)  # segments: two launches a pass
    leaves = [t.detach().clone().requires_grad_() for t in (x, g, s0)]

    def both():
        y, sT = la.gated_linear_recurrence(*leaves)
        return (y, sT, *torch.autograd.grad([y, sT], leaves, [dy, ds]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(leaves[0]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both()):
            assert torch.equal(a, b)


def test_empty():
    z = torch.zeros(2, 0, 8, device=DEV)
    s0 = torch.randn(2, 8, device=DEV)
    y, sT = la.gated_linear_recurrence(z, z, s0)
    assert y.shape == (2, 0, 8) and torch.equal(sT, s0)
    leaf = s0.clone().requires_grad_()
    y, sT = la.gated_linear_recurrence(z, z, leaf)
    assert torch.equal(torch.autograd.grad(sT.sum(), leaf)[0], torch.ones_like(s0))
    y, sT = la.gated_linear_recurrence(torch.zeros(0, 5, 8, device=DEV), torch.zeros(0, 5, 8, device=DEV))
    assert y.shape == (0, 5, 8) and sT.shape == (0, 8)
    y, s = la.gated_linear_recurrence_step(torch.zeros(0, 8, device=DEV), torch.zeros(0, 8, device=DEV), torch.zeros(0, 8, device=DEV))
    assert y.shape == (0, 8)


def test_refusals():
    x, g, s0, _, _ = _inputs(2, 5, 8, "f32", "f32", rows=2)
    for bad in (lambda: la.gated_linear_recurrence(x, g[:, :4]), lambda: la.gated_linear_recurrence(x, g, s0[:1]), lambda: la.gated_linear_recurrence(x[0], g[0]),
                lambda: la.gated_linear_recurrence(x.half(), g), lambda: la.gated_linear_recurrence(x, g, cu_seqlens=[0, 5]),
                lambda: la.gated_linear_recurrence(x, g.cpu()), lambda: la.gated_linear_recurrence(x, g.int()),
                lambda: la.gated_linear_recurrence_step(x[:, 0], g[:, 0], s0[:1]), lambda: la.gated_linear_recurrence_step(x[:, 0], g[:, 0], s0.bfloat16(), inplace=True)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        la.gated_linear_recurrence(x[:1], g[:1], cu_seqlens=[0, 4])
