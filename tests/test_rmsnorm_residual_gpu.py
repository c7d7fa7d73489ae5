"""rmsnorm_residual against its formulas in float64, with elementwise bounds that are carried through the formulas.

Bounds.  ``Num`` holds a value and a bound of its float32 error, u = 2^-24: a product adds |a| e_b + |b| e_a + u |ab|, a sum e_a + e_b +
u |a + b|, a sum of many terms the terms' bounds and u times its depth (additions in a row that one term passes through) times the sum
of magnitudes, 1 / sqrt half the relative error of its argument and one unit in the last place (2 u), the sigmoid s (1 - s) e + u (4 +
2 |z|) s (an exponential good to a unit, its scaled argument, a sum and a reciprocal).  Inputs are exact.  An output of type t is
rounded once: eps_t / 2 of its value."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
DEPTH = 64  # of a sum over a row: 16 columns a thread in a row, six levels in a wave, eight waves


class Num:
    def __init__(self, v, e=None):
        self.v = np.asarray(v, np.float64)
        self.e = np.zeros_like(self.v) if e is None else e

    def __add__(self, o):
        o = o if isinstance(o, Num) else Num(o)
        v = self.v + o.v
        return Num(v, self.e + o.e + U * np.abs(v))

    def __sub__(self, o):
        return self + Num(-o.v, o.e)

    def __mul__(self, o):
        o = o if isinstance(o, Num) else Num(o)
        v = self.v * o.v
        return Num(v, np.abs(self.v) * o.e + np.abs(o.v) * self.e + self.e * o.e + U * np.abs(v))

    def total(self, axis, depth):
        return Num(self.v.sum(axis, keepdims=axis == 1), (self.e + depth * U * np.abs(self.v)).sum(axis, keepdims=axis == 1))

    def rsqrt(self):
        v = 1 / np.sqrt(self.v)
        return Num(v, 0.5 * self.e / self.v * v + 3 * U * v)

    def sigmoid(self):
        s = 1 / (1 + np.exp(-self.v))
        return Num(s, s * (1 - s) * self.e + U * (4 + 2 * np.abs(self.v)) * s)


def _mean(a, d):
    return a.total(1, DEPTH) * (1.0 / d)


def _reference(x, r, w, post, gate, scale, dz, do):
    rows, d = x.shape
    one = Num(np.ones(d))
    X, c = Num(x), Num(np.broadcast_to(scale, (d,)))
    p = Num(post) if post is not None else one
    rho = (_mean(X * X, d) + EPS).rsqrt() if post is not None else Num(np.ones((rows, 1)))
    s = Num(gate).sigmoid() if gate is not None else Num(np.ones_like(x))
    xn, cp = X * rho, c * p
    R = xn * cp * s
    if r is not None:
        R = Num(r) + R
    out = {"r": R}
    D = Num(do)
    if w is not None:
        W, dZ = Num(w), Num(dz)
        rho2 = (_mean(R * R, d) + EPS).rsqrt()
        out["z"] = R * rho2 * W
        m = _mean(dZ * W * R, d) * rho2 * rho2
        D = D + rho2 * (dZ * W - R * m)
        out["dw"] = (dZ * R * rho2).total(0, rows + 16)
    if r is not None:
        out["dr"] = D
    both = (D * s * xn).total(0, rows + 16)
    V = D * cp * s
    m = _mean(V * X, d) * rho * rho if post is not None else Num(np.zeros((rows, 1)))
    out["dx"] = rho * (V - X * m)
    if gate is not None:
        out["dgate"] = V * xn * (Num(np.ones_like(x)) - s)
    if post is not None:
        out["dpost"] = both * c
    out["dscale"] = both * p
    return out


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _within(got, ref, what):
    eps = torch.finfo(got.dtype).eps / 2
    got, tol = _np(got), ref.e * (1 + 2 * eps) + eps * np.abs(ref.v) + 1e-37
    worst = np.abs(got - ref.v) / tol
    assert got.shape == ref.v.shape and np.all(worst <= 1), f"{what}: {worst.max():.2f} of the bound at {np.unravel_index(worst.argmax(), worst.shape)}"


CONFIGS = {  # post, gate, scale, residual, weight
    "all": (True, True, "channels", True, True),
    "number": (True, True, 0.7, True, True),
    "before": (False, False, 1.0, True, True),
    "channels": (False, False, "channels", True, True),
    "first": (False, False, 1.0, False, True),
    "last": (True, False, 0.5, True, False),
    "gated": (False, True, 1.0, False, True),
}


def _inputs(rows, d, dtype, r_dtype, config, seed=0):
    post, gate, scale, residual, weight = CONFIGS[config]
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, dt=torch.float32, std=1.0: (torch.randn(*s, generator=g) * std).to(DEV, dt)
    dt, rt = DT[dtype], DT[r_dtype]
    return dict(x=n(rows, d, dt=dt), residual=n(rows, d, dt=rt, std=2.0) if residual else None, weight=1 + n(d, std=0.3) if weight else None,
                post_weight=1 + n(d, std=0.3) if post else None, gate=n(rows, d, dt=dt, std=2.0) if gate else None,
                scale=0.5 + n(d, std=0.2) if scale == "channels" else scale), n(rows, d, dt=dt), n(rows, d, dt=rt if residual else dt)


def _check(t, dz, do):
    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if isinstance(v, torch.Tensor)}
    z, r = la.rmsnorm_residual(**{**t, **leaves}, eps=EPS)
    with torch.no_grad():
        z2, r2 = la.rmsnorm_residual(**t, eps=EPS)
    assert torch.equal(r, r2) and (z is None) == (z2 is None) == (t["weight"] is None)
    assert r.dtype == (t["x"] if t["residual"] is None else t["residual"]).dtype
    outs, cots = ([r], [do]) if z is None else ([z, r], [dz, do])
    if z is not None:
        assert torch.equal(z, z2) and z.dtype == t["x"].dtype
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), cots)))
    ref = _reference(*(_np(t[k]) if not isinstance(t[k], float) else t[k] for k in ("x", "residual", "weight", "post_weight", "gate", "scale")), _np(dz), _np(do))
    _within(r, ref["r"], "r")
    if z is not None:
        _within(z, ref["z"], "z")
    for k, name in (("x", "dx"), ("residual", "dr"), ("weight", "dw"), ("post_weight", "dpost"), ("gate", "dgate"), ("scale", "dscale")):
        if k in grads:
            _within(grads[k], ref[name], name)


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (3, 64), (7, 33), (4, 512), (9, 1000), (2, 1024), (5, 1032), (33, 2048), (5, 2050), (3, 4096), (2, 5001), (2, 8192), (1, 8191)])
def test_widths(rows, d, types):
    _check(*_inputs(rows, d, *types, "all"))


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("config", sorted(CONFIGS))
@pytest.mark.parametrize("rows,d", [(6, 72), (10, 2048), (3, 2056)])
def test_configurations(rows, d, config, types):
    _check(*_inputs(rows, d, *types, config, seed=1))


@pytest.mark.parametrize("types", [("bf16", "f32"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("rows,d", [(3100, 40), (1600, 1088)])
def test_many_rows(rows, d, types):
    """More rows than workgroups of the backward pass: every one goes through several."""
    _check(*_inputs(rows, d, *types, "all", seed=2))


def test_leading_dimensions_strides_and_types_of_parameters():
    t, dz, do = _inputs(12, 64, "bf16", "f32", "all")
    z, r = la.rmsnorm_residual(**t)
    shaped = {k: v.view(3, 4, 64) if v.dim() == 2 else v for k, v in t.items()}
    z3, r3 = la.rmsnorm_residual(**shaped)
    assert torch.equal(z3.view(12, 64), z) and torch.equal(r3.view(12, 64), r)
    wide = torch.cat([t["gate"], t["x"]], 1)
    zs, rs = la.rmsnorm_residual(**{**t, "x": wide[:, 64:], "gate": wide[:, :64], "residual": t["residual"].t().contiguous().t()})
    assert torch.equal(zs, z) and torch.equal(rs, r)
    off = torch.empty(12 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(12, 64).copy_(t["x"])  # rows that start beside a 16-byte boundary
    zo, _ = la.rmsnorm_residual(**{**t, "x": off})
    assert torch.allclose(zo.float(), z.float(), rtol=1e-2, atol=1e-5)
    half = {k: (v.bfloat16() if v.dim() == 1 else v).detach().requires_grad_() for k, v in t.items()}
    zh, rh = la.rmsnorm_residual(**half)
    grads = torch.autograd.grad([zh, rh], list(half.values()), [dz, do])
    assert all(g.dtype == v.dtype for g, v in zip(grads, half.values()))


def test_one_output_alone():
    t, dz, do = _inputs(20, 200, "f32", "f32", "all")
    leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
    z, r = la.rmsnorm_residual(**leaves)
    both = torch.autograd.grad([z, r], list(leaves.values()), [dz, do], retain_graph=True)
    by_z = torch.autograd.grad(z, list(leaves.values()), dz, retain_graph=True)
    by_r = torch.autograd.grad(r, list(leaves.values()), do, allow_unused=True)
    for k, a, b, c in zip(leaves, both, by_z, by_r):
        assert torch.allclose(a, b + (0 if c is None else c), rtol=1e-4, atol=1e-4 * float(a.abs().max())), k


def test_rows_keep_to_themselves():
    """A row with a NaN leaves every other row's outputs and row gradients alone."""
    t, dz, do = _inputs(40, 2048, "bf16", "f32", "all")
    z, r = la.rmsnorm_residual(**t)
    bad = {**t, "x": t["x"].clone()}
    bad["x"][17, 3] = float("nan")
    leaves = {k: v.detach().requires_grad_() for k, v in bad.items()}
    z2, r2 = la.rmsnorm_residual(**leaves)
    dx, dr = torch.autograd.grad([z2, r2], [leaves["x"], leaves["residual"]], [dz, do])
    rest = torch.arange(40, device=DEV) != 17
    assert torch.equal(z2[rest], z[rest]) and torch.equal(r2[rest], r[rest]) and bool(torch.isnan(z2[17]).all())
    assert bool(torch.isfinite(dx[rest]).all()) and bool(torch.isfinite(dr[rest]).all())


def test_gradients_against_differences():
    """Central differences in float32; the remainder of second order is step^2 of a third derivative of order one, the loss's rounding
    1e-6 over the step: together below one percent of the sum of magnitudes."""
    t, dz, do = _inputs(3, 24, "f32", "f32", "all", seed=4)
    leaves = {k: v.detach().requires_grad_() for k, v in t.items()}

    def loss(a):
        z, r = la.rmsnorm_residual(**a)
        return (z * dz).double().sum() + (r * do).double().sum()

    grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    g = torch.Generator().manual_seed(9)
    for k, v in t.items():
        dirn, step = torch.randn(v.shape, generator=g).to(DEV), 1e-2
        diff = (loss({**t, k: v + step * dirn}) - loss({**t, k: v - step * dirn})) / (2 * step)
        assert abs(float(diff - (grads[k].double() * dirn).sum())) < 1e-2 * float((grads[k].double() * dirn).abs().sum()), k


def test_repeats_bit_for_bit_and_replays():
    t, dz, do = _inputs(900, 520, "bf16", "f32", "all")
    leaves = {k: v.detach().clone().requires_grad_() for k, v in t.items()}

    def both():
        z, r = la.rmsnorm_residual(**leaves)
        return (z, r, *torch.autograd.grad([z, r], list(leaves.values()), [dz, do]))

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
            leaves["x"].copy_(torch.randn_like(leaves["x"]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both()))


def test_more_rows_than_one_direction_of_a_launch():
    rows = 2 ** 26 + 5  # of 64 threads: more than 2^32
    x = torch.zeros(rows, 8, dtype=torch.bfloat16, device=DEV)
    x[-7:] = torch.randn(7, 8, generator=torch.Generator().manual_seed(5)).to(DEV, torch.bfloat16)
    w = torch.ones(8, device=DEV)
    leaves = [t.detach().requires_grad_() for t in (x, x[-7:])]
    whole, few = (la.rmsnorm_residual(t, None, w) for t in leaves)
    assert all(torch.equal(a[-7:], b) and not bool(a[:-7].any()) for a, b in zip(whole, few))
    dz = torch.ones_like(whole[0])
    dx, ds = torch.autograd.grad(whole[0], leaves[0], dz)[0], torch.autograd.grad(few[0], leaves[1], dz[-7:])[0]
    assert torch.equal(dx[-7:], ds)


def test_empty():
    w = torch.ones(32, device=DEV, requires_grad=True)
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    z, r = la.rmsnorm_residual(x, None, w)
    assert z.shape == r.shape == (0, 32)
    gx, gw = torch.autograd.grad(z.sum(), [x, w])
    assert gx.shape == (0, 32) and bool((gw == 0).all())


def test_refusals():
    x, w = torch.randn(4, 32, device=DEV), torch.ones(32, device=DEV)
    for bad in (lambda: la.rmsnorm_residual(x, x[:2], w), lambda: la.rmsnorm_residual(x, x.bfloat16(), w), lambda: la.rmsnorm_residual(x.half(), None, w),
                lambda: la.rmsnorm_residual(x, x, w[:8]), lambda: la.rmsnorm_residual(x, x, w, gate=x[:, :8]), lambda: la.rmsnorm_residual(x, x, w, scale=w[:1]),
                lambda: la.rmsnorm_residual(x, x.cpu(), w), lambda: la.rmsnorm_residual(x, x, w.int()),
                lambda: la.rmsnorm_residual(torch.zeros(1, 8193, device=DEV), None, torch.ones(8193, device=DEV))):
        with pytest.raises(RuntimeError):
            bad()
