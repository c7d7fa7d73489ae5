"""layer_norm against its formulas in float64, with elementwise bounds that are carried through the formulas (``Num`` of
test_rmsnorm_residual_gpu.py: a value and a bound of its float32 error).  An output of type t is rounded once: eps_t / 2 of its value."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la
from test_rmsnorm_residual_gpu import DEPTH, DEV, DT, EPS, Num, _np, _within

pytestmark = pytest.mark.gpu


def _mean(a, d):
    return a.total(1, DEPTH) * Num(np.float64(1.0 / d), np.float64(2.0 ** -24 / d))


def _reference(x, w, b, dy, heads):
    """x, dy [rows, d]; w, b [heads, d] or None"""
    rows, d = x.shape
    per = lambda t, none: Num(np.tile(t, (rows // heads, 1)) if t is not None else np.full((rows, d), none))
    X, W, dY = Num(x), per(w, 1.0), Num(dy)
    xc = X - _mean(X, d)
    rho = (_mean(xc * xc, d) + EPS).rsqrt()
    h = xc * rho
    out = {"y": h * W + per(b, 0.0)}
    u = dY * W
    out["dx"] = rho * (u - _mean(u, d) - xc * (_mean(u * xc, d) * rho * rho))

    def over_rows(t):
        v, e = (a.reshape(rows // heads, heads, d) for a in (t.v, t.e))
        return Num(v.sum(0), (e + (rows // heads + 16) * 2.0 ** -24 * np.abs(v)).sum(0))

    out["dw"], out["db"] = over_rows(dY * h), over_rows(dY)
    return out


def _inputs(shape, dtype, weights="both", heads=1, seed=0, offset=0.7):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, dt=torch.float32, std=1.0: (torch.randn(*s, generator=g) * std).to(DEV, dt)
    ws = (heads, shape[-1]) if heads > 1 else shape[-1:]
    x = (torch.randn(*shape, generator=g) * 2 + offset).to(DEV, DT[dtype])
    return x, 1 + n(*ws, std=0.3) if weights in ("both", "weight") else None, n(*ws, std=0.5) if weights in ("both", "bias") else None, n(*shape, dt=DT[dtype])


def _check(x, w, b, dy, heads=1):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = la.layer_norm(*leaves, EPS)
    with torch.no_grad():
        assert torch.equal(la.layer_norm(x, w, b, EPS), y)
    assert y.shape == x.shape and y.dtype == x.dtype
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    flat = lambda t: _np(t).reshape(-1, x.shape[-1])
    ref = _reference(flat(x), None if w is None else flat(w), None if b is None else flat(b), flat(dy), heads)
    _within(y.reshape(-1, x.shape[-1]), ref["y"], "y")
    for t, name in zip(leaves, ("dx", "dw", "db")):
        if t is not None:
            g = next(grads)
            assert g.shape == t.shape and g.dtype == t.dtype
            _within(g.reshape(-1, x.shape[-1]), ref[name], name)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (5, 30), (3, 64), (7, 33), (70, 65), (9, 128), (21, 200), (4, 512), (9, 1000), (2, 1024), (5, 1032), (33, 2048), (5, 2050),
                                    (3, 4096), (2, 5001), (2, 8192), (1, 8191)])
def test_widths(rows, d, dtype):
    _check(*_inputs((rows, d), dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("weights", ["none", "weight", "bias"])
@pytest.mark.parametrize("rows,d", [(6, 72), (10, 2048), (300, 64)])
def test_weights_that_are_absent(rows, d, weights, dtype):
    _check(*_inputs((rows, d), dtype, weights, seed=1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,heads,d", [(1, 3, 64), (50, 5, 128), (7, 16, 33), (33, 2, 256), (9, 3, 520), (3, 2, 2048), (900, 4, 64), (2, 800, 16)])
def test_weights_for_each_head(rows, heads, d, dtype):
    _check(*_inputs((rows, heads, d), dtype, heads=heads, seed=2), heads=heads)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,d", [(140000, 64), (3100, 40), (70000, 136), (1600, 1088)])
def test_many_rows(rows, d, dtype):
    """Several rows a thread in the forward pass, several turns of every workgroup in the backward pass."""
    _check(*_inputs((rows, d), dtype, seed=3))


def test_a_mean_far_from_zero():
    """The variance is a sum of squared differences: rows around 10000 keep their seven digits."""
    x, w, b, dy = _inputs((40, 768), "f32", seed=4, offset=1e4)
    _check(x, w, b, dy)
    want = torch.nn.functional.layer_norm(x.double(), (768,), w.double(), b.double(), EPS)
    assert float((la.layer_norm(x, w, b, EPS).double() - want).abs().max()) < 3e-3  # a unit of 1e4 is 1e-3; the rows' deviation is 2


def test_constant_rows():
    x = torch.full((5, 130), 3.0, device=DEV, requires_grad=True)
    b = torch.randn(130, device=DEV)
    y = la.layer_norm(x, None, b)
    assert torch.allclose(y, b.expand(5, 130), atol=1e-2)  # (3 - mean) is at most a unit or two of 3, and 1 / sqrt(eps) = 316
    assert bool(torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all())


def test_leading_dimensions_strides_and_types_of_parameters():
    x, w, b, dy = _inputs((12, 64), "bf16")
    y = la.layer_norm(x, w, b)
    assert torch.equal(la.layer_norm(x.view(3, 4, 64), w, b).view(12, 64), y)
    assert torch.equal(la.layer_norm(torch.cat([x, x], 1)[:, 64:], w, b), y)
    assert torch.equal(la.layer_norm(x.view(3, 4, 64).transpose(0, 1), w, b).transpose(0, 1).reshape(12, 64), y)
    off = torch.empty(12 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(12, 64).copy_(x)  # rows that start beside a 16-byte boundary
    assert torch.allclose(la.layer_norm(off, w, b).float(), y.float(), rtol=1e-2, atol=1e-2)
    assert torch.equal(la.layer_norm(x[0], w, b), y[0])
    half = [t.bfloat16().detach().requires_grad_() for t in (x, w, b)]
    assert all(g.dtype == torch.bfloat16 for g in torch.autograd.grad(la.layer_norm(*half), half, dy))
    wide = dy[:, :1].expand(12, 64)  # a broadcast gradient
    leaf = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(la.layer_norm(leaf, w, b), leaf, wide)[0], torch.autograd.grad(la.layer_norm(leaf, w, b), leaf, wide.contiguous())[0])


@pytest.mark.parametrize("shape,heads", [((40, 2048), 1), ((40, 4, 32), 4), ((64, 48), 1)])
def test_rows_keep_to_themselves(shape, heads):
    """A row with a NaN leaves every other row's outputs and row gradients alone."""
    x, w, b, dy = _inputs(shape, "bf16", heads=heads)
    y = la.layer_norm(x, w, b)
    bad = x.clone()
    bad[17].view(-1)[3] = float("nan")
    leaf = bad.requires_grad_()
    y2 = la.layer_norm(leaf, w, b)
    dx, = torch.autograd.grad(y2, leaf, dy)
    rest = torch.ones(shape[:-1], dtype=torch.bool, device=DEV)
    rest[(17, 0) if heads > 1 else 17] = False
    assert torch.equal(y2[rest], y[rest]) and bool(torch.isnan(y2[~rest]).all()) and bool(torch.isfinite(dx[rest]).all())


def test_gradients_against_differences():
    """Central differences in float32, as in test_rmsnorm_residual_gpu.py: below one percent of the sum of magnitudes."""
    x, w, b, dy = _inputs((3, 2, 24), "f32", heads=2, seed=4)
    t = {"x": x, "weight": w, "bias": b}
    leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
    loss = lambda a: (la.layer_norm(**a) * dy).double().sum()
    grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    g = torch.Generator().manual_seed(9)
    for k, v in t.items():
        dirn, step = torch.randn(v.shape, generator=g).to(DEV), 1e-2
        diff = (loss({**t, k: v + step * dirn}) - loss({**t, k: v - step * dirn})) / (2 * step)
        assert abs(float(diff - (grads[k].double() * dirn).sum())) < 1e-2 * float((grads[k].double() * dirn).abs().sum()), k


def test_repeats_bit_for_bit_and_replays():
    x, w, b, dy = _inputs((900, 8, 72), "bf16", heads=8)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]

    def both():
        y = la.layer_norm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

    assert all(torch.equal(a, c) for a, c in zip(both(), both()))
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
            leaves[0].copy_(torch.randn_like(leaves[0]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, both()))


def test_refused_while_a_graph_of_the_leaf_is_alive():
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    alive = la.layer_norm(x)
    graph, keep = torch.cuda.CUDAGraph(), torch.zeros(8, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        keep.add_(1)
        with pytest.raises(RuntimeError, match="alive"):
            la.layer_norm(x)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((keep == 1).all()) and bool(torch.isfinite(alive).all())


def test_rows_beyond_two_to_the_31_elements():
    rows = 2 ** 20 + 3
    x = torch.zeros(rows, 2048, dtype=torch.bfloat16, device=DEV)
    x[-5:] = torch.randn(5, 2048, generator=torch.Generator().manual_seed(5)).to(DEV, torch.bfloat16)
    leaf, few = x.requires_grad_(), x.detach()[-5:].clone().requires_grad_()
    y, ys = la.layer_norm(leaf), la.layer_norm(few)
    assert torch.equal(y[-5:], ys) and not bool(y[:-5].any())
    dx, = torch.autograd.grad(y, leaf, y.detach())
    assert torch.equal(dx[-5:], torch.autograd.grad(ys, few, ys.detach())[0])


def test_empty():
    w, b = torch.ones(32, device=DEV, requires_grad=True), torch.ones(32, device=DEV, requires_grad=True)
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    gx, gw, gb = torch.autograd.grad(la.layer_norm(x, w, b).sum(), [x, w, b])
    assert gx.shape == (0, 32) and bool((gw == 0).all()) and bool((gb == 0).all())


def test_refusals():
    x, w = torch.randn(4, 32, device=DEV), torch.ones(32, device=DEV)
    for bad in (lambda: la.layer_norm(x.half(), w), lambda: la.layer_norm(x, w[:8]), lambda: la.layer_norm(x, w, w[:8]), lambda: la.layer_norm(x, w.cpu()),
                lambda: la.layer_norm(x, w.int()), lambda: la.layer_norm(x, torch.ones(3, 32, device=DEV)), lambda: la.layer_norm(x, w, torch.ones(4, 32, device=DEV)),
                lambda: la.layer_norm(torch.zeros(1, 8193, device=DEV)), lambda: la.layer_norm(x, w, None, float("nan")), lambda: la.layer_norm(x, w, None, -1.0),
                lambda: la.layer_norm(torch.zeros(3, 0, device=DEV)), lambda: la.layer_norm(torch.tensor(1.0, device=DEV)), lambda: la.layer_norm(x.cpu(), w)):
        with pytest.raises(RuntimeError):
            bad()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            la.layer_norm(torch.autograd.forward_ad.make_dual(x, x), w)
