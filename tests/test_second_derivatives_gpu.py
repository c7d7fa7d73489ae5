"""Second derivatives, which the backward kernels do not have: whatever asks for one is told so, whatever does not is not disturbed."""
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _decay(leaves):
    return la.decay_linear_attention(*leaves)[0]


def _token(leaves):
    q, k, v, g, s = leaves
    return la.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g, s[:, :, :64])[0]


def _norm(leaves):
    return la.layer_norm(leaves[0], leaves[1], leaves[2])


def _leaves(op):
    gen = torch.Generator().manual_seed(1)
    if op is _norm:
        shapes = [(5, 64), (64,), (64,)]
    else:
        shapes = [(1, 2, 20, 64)] * 3 + [(2,)] + ([(1, 2, 64, 64)] if op is _token else [])
    return [(torch.randn(s, generator=gen) * (-1 if len(s) == 1 and op is not _norm else 1)).to(DEV).requires_grad_() for s in shapes]


@pytest.mark.parametrize("name,op", [("decay_linear_attention", _decay), ("decay_linear_attention", _token), ("layer_norm", _norm)], ids=["decay", "token", "norm"])
def test_second_derivatives_are_refused(name, op):
    leaves = _leaves(op)
    want = torch.autograd.grad(op(leaves).square().sum(), leaves)
    got = torch.autograd.grad(op(leaves).square().sum(), leaves, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape
    for i, g in enumerate(got):
        with pytest.raises(NotImplementedError, match=f"{name} has no second derivative"):
            torch.autograd.grad(g.sum(), leaves[i], retain_graph=True)
    # a penalty on the gradient beside terms that have derivatives: not half of one, whoever asks and however
    for ask in (lambda loss: loss.backward(retain_graph=True), lambda loss: torch.autograd.grad(loss, leaves[0], retain_graph=True), lambda loss: torch.autograd.grad(loss, leaves[1], retain_graph=True)):
        with pytest.raises(NotImplementedError, match="second derivative"):
            ask(leaves[0].square().sum() + leaves[1].square().sum() + got[0].square().sum())


def test_derivatives_with_respect_to_what_came_in_are_refused():
    """The gradient is linear in the incoming one, whose graph may be all that is asked for."""
    x, dy = torch.randn(5, 64, device=DEV, requires_grad=True), torch.randn(5, 64, device=DEV, requires_grad=True)
    dx = torch.autograd.grad(la.layer_norm(x), x, dy, create_graph=True)[0]
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(dx.sum(), dy)


def test_gradients_kept_for_a_graph_that_nobody_differentiates():
    leaves = _leaves(_norm)
    _norm(leaves).sum().backward(create_graph=True)
    assert bool(torch.isfinite(leaves[0].grad).all()) and leaves[0].grad.shape == leaves[0].shape
    for x in leaves:
        x.grad = None
