"""decay_linear_attention where there is little or nothing: no rows, no tokens, a gradient that nobody's value reaches."""
import ctypes as C

import pytest
import torch

import linearnexus_amd as la
from linearnexus_amd import _lib
from test_decay_attention_gpu import CHUNK, DT, _close, _formulas, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_decay_for_each_head_has_a_gradient_of_zeros_without_rows():
    g = torch.full((3,), -0.5, device=DEV, requires_grad=True)
    q, s0 = torch.zeros(0, 3, 5, 64, device=DEV, requires_grad=True), torch.zeros(0, 3, 64, 64, device=DEV)
    o, s = la.decay_linear_attention(q, q, q, g)
    assert bool((torch.autograd.grad(o.sum() + s.sum(), g)[0] == 0).all())
    o, s = la.decay_linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], g, s0)
    assert bool((torch.autograd.grad(o.sum() + s.sum(), g)[0] == 0).all())


def test_the_c_call_writes_zeros_without_rows():
    d_g = torch.full((5,), float("nan"), device=DEV)
    a = _lib.DecayArgs(B=0, H=3, T=5, dk=64, dv=64, dtype=_lib.LNX_F32, g_per_head=1, scale=1.0)
    a.d_g = C.c_void_p(d_g.data_ptr())
    assert _lib.load().lnx_decay_bwd(a, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert bool((d_g[:3] == 0).all()) and bool(d_g[3:].isnan().all())


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_rows_without_tokens_have_gradients(packed, per_head):
    """The last state is the initial one: its gradient passes through, the others are empty, or zeros for each head."""
    rows = 3 if packed else 2
    z = torch.zeros(1 if packed else 2, 2, 0, 64, device=DEV, requires_grad=True)
    g = torch.zeros(2 if per_head else (z.shape[0], 2, 0), device=DEV, requires_grad=True)
    s0, ds = (torch.randn(rows, 2, 64, 64, device=DEV) for _ in range(2))
    s0.requires_grad_()
    o, s = la.decay_linear_attention(z, z, z, g, None, s0, cu_seqlens=[0] * 4 if packed else None)
    assert torch.equal(s, s0) and o.shape == z.shape
    dz, dg, d0 = torch.autograd.grad([o, s], [z, g, s0], [torch.zeros_like(o), ds])
    assert dz.shape == z.shape and dg.shape == g.shape and bool((dg == 0).all()) and torch.equal(d0, ds)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("T,at", [(1, 0), (100, 0), (100, 63), (100, 99), (150, 70), (1100, 0), (1100, 300), (1100, 1099), (2600, 1700)])
def test_gates_gradients_beside_values_that_are_not_finite(T, at, which, per_head, dtype):
    """dg_t = e^g <dS_t, S_{t-1}> takes keys and values of earlier tokens and queries and gradients of t and later ones: the others' dg is what it is
    without the value, within the bound of the terms that it is summed from; other heads' is the same bit for bit.  (1100 tokens and more: in segments.)"""
    for value in (float("nan"), float("inf")):
        t, do, ds = _inputs(1, 2, T, 64, 64, dtype, per_head=per_head, decay=0.1, seed=41)
        leaves = {n: x.detach().requires_grad_() for n, x in t.items()}
        bad = {**{n: t[n].clone() for n in ("q", "k", "v")}, "do": do.clone()}
        bad[which][0, 1, at, 5] = value
        grads = []
        for x in ({**t, "do": do}, bad):
            g = t["g"].detach().requires_grad_()
            o, sT = la.decay_linear_attention(x["q"], x["k"], x["v"], g, None, t["s0"])
            grads.append(torch.autograd.grad([o, sT], g, [x["do"], ds])[0])
        E = (2.0 ** -15 if dtype == "bf16" else 0.0) + (T + 192) * 2.0 ** -23 + 17 * 2.0 ** -20
        x = [t[n][0, 1].double() for n in ("q", "k", "v")]
        gg = (t["g"][1].expand(T) if per_head else t["g"][0, 1]).double()
        back = [do[0, 1].double(), ds[0, 1].double()]
        ref = _formulas(*x, gg, t["s0"][0, 1].double(), 64 ** -0.5, *back, CHUNK[DT[dtype]])["dg"]
        mag = _formulas(*(y.abs() for y in x), gg, t["s0"][0, 1].double().abs(), 64 ** -0.5, *(y.abs() for y in back), CHUNK[DT[dtype]])["dg sums"]
        tokens = torch.arange(T, device=DEV)
        fine = tokens <= at if which in ("k", "v") else tokens > at
        if per_head:
            assert torch.equal(grads[0][0], grads[1][0])
            if bool(fine.all()):
                _close(grads[1][1], ref.sum(), (2 * E * mag).sum() + (T + 16) * 2.0 ** -23 * ref.abs().sum(), "dg")
            else:
                assert not bool(torch.isfinite(grads[1][1]))
        else:
            assert torch.equal(grads[0][0, 0], grads[1][0, 0])
            _close(grads[1][0, 1][fine], ref[fine], (2 * E * mag)[fine], "dg")
            assert not bool(torch.isfinite(grads[1][0, 1][~fine]).any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("at", [100, 1024, 2100, 2221])
def test_gates_gradients_beside_a_value_that_is_not_finite_in_a_long_row(at, dtype):
    """Heads enough that rows are walked whole: more tokens than are summed at a time."""
    H, T = 130, 2222
    t, do, ds = _inputs(1, H, T, 16, 16, dtype, state=False, decay=0.1, seed=42)
    v = t["v"].clone()
    v[0, 7, at, 3] = float("inf")
    grads = []
    for x in (t["v"], v):
        g = t["g"].detach().requires_grad_()
        o, sT = la.decay_linear_attention(t["q"], t["k"], x, g)
        grads.append(torch.autograd.grad([o, sT], g, [do, ds])[0][0])
    others = torch.arange(H, device=DEV) != 7
    assert torch.equal(grads[0][others], grads[1][others]) and not bool(torch.isfinite(grads[1][7, at + 1 :]).any())
    x = [t[n][0, 7].double() for n in ("q", "k", "v", "g")]
    back = [do[0, 7].double(), ds[0, 7].double()]
    zero = torch.zeros(16, 16, dtype=torch.float64, device=DEV)
    ref = _formulas(*x, zero, 0.25, *back, CHUNK[DT[dtype]])["dg"]
    mag = _formulas(*(y.abs() for y in x[:3]), x[3], zero, 0.25, *(y.abs() for y in back), CHUNK[DT[dtype]])["dg sums"]
    E = (2.0 ** -15 if dtype == "bf16" else 0.0) + (T + 96) * 2.0 ** -23 + 17 * 2.0 ** -20
    _close(grads[1][7, : at + 1], ref[: at + 1], (2 * E * mag)[: at + 1], "dg")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("loud", ["first", "second"])
def test_gates_gradients_of_a_quiet_half_beside_a_loud_one(loud, dtype):
    """One half's values are a thousand times the other's, a reset between them, in rows that are walked whole: the quiet half's dg is what it is alone.  By
    norms: at most nine roundings of a state for each chunk of 32, 3 2^-23 + (9 T / 32)^(1/2) 2^-24 < 2^-18 of it, twice that of dg, and as much again for its
    share in what the row's sums miss: 2^-16."""
    B, H, T, d = 2, 66, 4096, 16
    t, do, _ = _inputs(B, H, T, d, d, dtype, state=False, decay=0.002, seed=43)
    half = {"first": slice(0, T // 2), "second": slice(T // 2, T)}
    t["v"][:, :, half[loud]] *= 1000.0
    t["g"][:, :, T // 2] = -float("inf")
    g = t["g"].detach().requires_grad_()
    o, _ = la.decay_linear_attention(t["q"], t["k"], t["v"], g)
    got = torch.autograd.grad(o, g, do)[0]
    quiet = half["second" if loud == "first" else "first"]
    zero = torch.zeros(d, d, dtype=torch.float64, device=DEV)
    for b, h in ((0, 0), (0, 37), (1, 65)):
        x = [y[b, h, quiet].double() for y in (t["q"], t["k"], t["v"], t["g"])]
        x[3] = x[3].clamp_min(-60.0)  # (the reset is the first of the second half, whose own state is empty)
        want = _formulas(*x, zero, d ** -0.5, do[b, h, quiet].double(), zero, CHUNK[DT[dtype]])["dg"]
        off = float((got[b, h, quiet].double() - want).norm() / want.norm())
        assert off < 2.0 ** -16, f"{off:.2g}"


@pytest.mark.parametrize("T", [40, 1100])
def test_decode_steps_go_on_from_a_prompts_state_in_place(T):
    """The prompt's gradient needs its last state only where that has a gradient: otherwise a step may write over it, and its gradient is refused."""
    t, do, ds = _inputs(1, 2, T, 64, 64, "f32", seed=44)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    o, s = la.decay_linear_attention(*leaves)
    want = torch.autograd.grad(o, leaves, do, retain_graph=True)
    la.decay_linear_attention_step(*(t[n][:, :, 0] for n in ("q", "k", "v", "g")), s.detach(), inplace=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, leaves, do, retain_graph=True), want))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([o, s], leaves, [do, ds])
