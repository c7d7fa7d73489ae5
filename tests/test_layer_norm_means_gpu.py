"""layer_norm of rows whose mean is far from zero, against its formulas in float64.

Bounds as in test_layer_norm_gpu.py, but from the differences on.  The first mean is off by units of itself (below 0.1 for means of 10^5: 64 additions of 2^-24).  x less that is exact (both lie
within a factor of two of each other), and what the differences' own mean misses is a sum of them: (64 + 1) 2^-24 of their mean magnitude, however large x is, plus a rounding
of its subtraction."""
import numpy as np
import pytest
import torch

import linearnexus_amd as la
from test_layer_norm_gpu import _inputs, _mean
from test_rmsnorm_residual_gpu import DEPTH, DEV, EPS, U, Num, _np, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [1e4, -1e5])
@pytest.mark.parametrize("shape,heads", [((40, 768), 1), ((60, 4, 64), 4), ((9, 3, 33), 3), ((5, 5000), 1), ((3, 8192), 1), ((7, 1001), 1), ((9000, 40), 1)])
def test_rows_around_a_large_mean(shape, heads, offset):
    x, w, b, dy = _inputs(shape, "f32", heads=heads, seed=11, offset=offset)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = la.layer_norm(*leaves, EPS)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    d = shape[-1]
    X, dY = _np(x).reshape(-1, d), Num(_np(dy).reshape(-1, d))
    rows = X.shape[0]
    W, b_ = (Num(np.tile(_np(t).reshape(heads, d), (rows // heads, 1))) for t in (w, b))
    c = X - X.mean(1, keepdims=True)
    xc = Num(c, (DEPTH + 1) * U * (np.abs(c).mean(1, keepdims=True) + 0.1) + U * np.abs(c))
    rho = (_mean(xc * xc, d) + EPS).rsqrt()
    h, u = xc * rho, dY * W
    _within(y.reshape(-1, d), h * W + b_, "y")
    _within(dx.reshape(-1, d), rho * (u - _mean(u, d) - xc * (_mean(u * xc, d) * rho * rho)), "dx")
    for got, t, name in ((dw, dY * h, "dw"), (db, dY, "db")):
        v, e = (a.reshape(rows // heads, heads, d) for a in (t.v, t.e))
        _within(got.reshape(heads, d), Num(v.sum(0), (e + (rows // heads + 16) * U * np.abs(v)).sum(0)), name)


def test_constant_rows_are_the_bias():
    """Differences of a unit of 3 at the most, whose mean misses them by 65 2^-24: times 316 = 1 / sqrt(eps) less than 1e-9."""
    x = torch.full((5, 130), 3.0, device=DEV)
    b = torch.randn(130, device=DEV)
    assert bool(((la.layer_norm(x, None, b) - b).abs() <= 1e-9 + 2.0 ** -23 * b.abs()).all())


def test_rows_with_an_infinite_value_have_no_finite_one():
    x = torch.randn(4, 300, device=DEV)
    x[1, 7], x[2, 9] = float("inf"), float("nan")
    y = la.layer_norm(x)
    assert not bool(torch.isfinite(y[1:3]).any()) and torch.equal(y[[0, 3]], la.layer_norm(x[[0, 3]]))
