"""decay_linear_attention where there is little or nothing: no rows, no tokens, a gradient that nobody's value reaches."""
import ctypes as C

import pytest
import torch

import linearnexus_amd as la
from linearnexus_amd import _lib

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
