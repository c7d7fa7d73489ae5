"""The gated linear recurrence at its edges."""
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# -- recurrence: one token whose token stride says nothing ------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_token_of_a_sequence_first_batch(dtype):
    """[1, B, D] transposed: the stride over the one token is the whole batch, more than the kernels step over."""
    B, D = 520, 8192
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(1, B, D, generator=g).to(DEV, DT[dtype]).transpose(0, 1) for _ in range(2))
    decay = -torch.rand(1, B, D, generator=g).to(DEV).transpose(0, 1)
    s0 = torch.randn(B, D, generator=g).to(DEV)
    leaves = [t.detach().requires_grad_() for t in (x, decay, s0)]
    y, state = la.gated_linear_recurrence(*leaves)
    dx, dg, ds = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dx, dy)
    # float32 throughout: an exponential good to two units, its argument (at most 1) to one, products and a sum of half a unit each: below 8 u
    e, xd, dyd = torch.exp(decay[:, 0].double()), x[:, 0].double(), dy[:, 0].double()
    eps = torch.finfo(x.dtype).eps / 2
    for got, ref, mag, last in ((y[:, 0], e * s0 + xd, (e * s0).abs() + xd.abs(), eps), (state, e * s0 + xd, (e * s0).abs() + xd.abs(), 0),
                                (dg[:, 0], e * s0 * dyd, (e * s0 * dyd).abs(), 0), (ds, e * dyd, (e * dyd).abs(), 0)):
        assert bool(((got.double() - ref).abs() <= 2.0 ** -21 * mag + last * (ref.abs() + 2.0 ** -21 * mag) + 1e-36).all())
