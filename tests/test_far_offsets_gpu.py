"""Rows that lie more than 2^31 elements apart: offsets of the recurrence, the residual norm and attention are 64-bit."""
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
FAR = 2 ** 31 + 1024


@pytest.fixture(scope="module")
def memory():
    return torch.zeros(FAR + 2 ** 22, dtype=torch.bfloat16, device=DEV)


def _far(memory, shape, at, seed):
    """A [2, ...] view whose two rows are FAR elements apart, starting `at` elements in, filled with random values."""
    n = torch.Size(shape[1:]).numel()
    strides = torch.empty(shape[1:]).stride()
    view = memory.as_strided(shape, (FAR, *strides), at)
    view.copy_(torch.randn(shape, generator=torch.Generator().manual_seed(seed)))
    assert at + n <= 2 ** 22
    return view


def test_recurrence(memory):
    x, g = _far(memory, (2, 300, 64), 0, 0), _far(memory, (2, 300, 64), 2 ** 20, 1)
    g.copy_(-g.abs())
    for a, b in zip(la.gated_linear_recurrence(x, g), la.gated_linear_recurrence(x.contiguous(), g.contiguous())):
        assert torch.equal(a, b)
    leaves, near = ([t.detach().requires_grad_() for t in ts] for ts in ((x, g), (x.contiguous(), g.contiguous())))
    dy = _far(memory, (2, 300, 64), 2 ** 21, 2)
    want = torch.autograd.grad(la.gated_linear_recurrence(*near)[0], near, dy.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(la.gated_linear_recurrence(*leaves)[0], leaves, dy), want))


def test_attention(memory):
    q, k, v, do = (_far(memory, (2, h, 130, 64), i * 2 ** 20, i) for i, h in enumerate((4, 2, 2, 4)))
    outs = []
    for ts in ((q, k, v, do), tuple(t.contiguous() for t in (q, k, v, do))):
        leaves = [t.detach().requires_grad_() for t in ts[:3]]
        o = la.causal_attention(*leaves)
        outs.append((o, *torch.autograd.grad(o, leaves, ts[3])))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_attention_step(memory):
    kc, vc = _far(memory, (2, 2, 300, 64), 0, 5), _far(memory, (2, 2, 300, 64), 2 ** 20, 6)
    near = kc.contiguous(), vc.contiguous()
    q, k, v = (torch.randn(2, h, 64, device=DEV).bfloat16() for h in (4, 2, 2))
    lengths = torch.tensor([299, 40], dtype=torch.int32, device=DEV)
    assert torch.equal(la.causal_attention_step(q, k, v, kc, vc, lengths), la.causal_attention_step(q, k, v, *near, lengths))
    assert torch.equal(kc, near[0]) and torch.equal(vc, near[1])


def test_many_rows_of_the_residual_norm():
    rows, d = 2 ** 20 + 3, 2056  # 2.2e9 elements
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device=DEV)
    x[-5:] = torch.randn(5, d, device=DEV).bfloat16()
    w = torch.ones(d, device=DEV)
    z, r = la.rmsnorm_residual(x, None, w)
    zs, rs = la.rmsnorm_residual(x[-5:], None, w)
    assert torch.equal(z[-5:], zs) and torch.equal(r[-5:], rs) and not bool(z[:-5].any())


def test_a_result_of_more_than_2_31_elements():
    T, D = 2 ** 19 + 130, 4128
    x = torch.zeros(1, T, D, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device=DEV).expand(1, T, D)
    x[0, 7] = 1
    y, s = la.gated_linear_recurrence(x, g)
    assert bool((s == 1).all()) and bool((y[0, -3:] == 1).all()) and not bool(y[0, :7].any())
    del x, g, y, s
    x = torch.zeros(1, T, D, dtype=torch.bfloat16, device=DEV)
    x[0, 7] = 1
    x.requires_grad_()
    g = torch.zeros(1, T, 1, dtype=torch.bfloat16, device=DEV).expand(1, T, D).requires_grad_()
    y = la.gated_linear_recurrence(x, g)[0]
    dy = torch.zeros_like(x)
    dy[0, -2] = 1
    dx, dg = torch.autograd.grad(y, (x, g), dy)
    assert bool((dx[0, :-1] == 1).all()) and not bool(dx[0, -1].any())
    assert bool((dg[0, 8:-1] == 1).all()) and not bool(dg[0, :8].any()) and not bool(dg[0, -1].any())


def test_attention_of_more_than_2_31_elements():
    H, d, lens = 17, 128, [128] * 8190 + [200]
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    T = cu[-1]
    q, do = (torch.randn(1, H, T, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(1, 1, T, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    assert q.numel() > 2 ** 31
    outs = []
    for lo in (0, cu[-2]):
        leaves = [t[:, :, lo:].detach().requires_grad_() for t in (q, k, v)]
        o = la.causal_attention(*leaves, cu_seqlens=cu if lo == 0 else None)
        outs.append([t[:, :, -200:] for t in (o, *torch.autograd.grad(o, leaves, do[:, :, lo:]))])
    # the same sums, of the lone sequence perhaps split between workgroups: both round operands and results to 2^-8 of themselves
    for a, b in zip(*outs):
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 2 ** -6
