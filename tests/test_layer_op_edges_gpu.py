"""The gated linear recurrence and the residual norm at their edges; captured passes and in-place steps of both and of attention."""
import pytest
import torch

import linearnexus_amd as la
from test_rmsnorm_residual_gpu import _np as _npy, _reference as _norm_reference, _within as _norm_within

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


# -- residual norm: a gate in float32 beside bfloat16 ------------------------------------------------------------------

@pytest.mark.parametrize("r_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,d", [(5, 33), (7, 64), (3, 512), (9, 1000), (4, 1024), (6, 2048), (3, 3001), (2, 4096), (2, 8192), (1500, 264)])
def test_gate_keeps_its_type(rows, d, r_dtype):
    """Neither the gate nor its gradient is rounded to x's type: both are what the formula gives, in float32."""
    g = torch.Generator().manual_seed(rows + d)
    n = lambda *s, t=torch.float32, std=1.0: (torch.randn(*s, generator=g) * std).to(DEV, t)
    x, r, gate, w, post = n(rows, d, t=torch.bfloat16), n(rows, d, t=DT[r_dtype], std=2.0), n(rows, d, std=2.0), 1 + n(d, std=0.3), 1 + n(d, std=0.3)
    dz, do = n(rows, d, t=torch.bfloat16), n(rows, d, t=DT[r_dtype])
    leaves = [t.detach().requires_grad_() for t in (x, r, w, post, gate)]
    z, out = la.rmsnorm_residual(leaves[0], leaves[1], leaves[2], leaves[3], leaves[4], 0.7)
    grads = torch.autograd.grad([z, out], leaves, [dz, do])
    ref = _norm_reference(_npy(x), _npy(r), _npy(w), _npy(post), _npy(gate), 0.7, _npy(dz), _npy(do))
    _norm_within(z, ref["z"], "z")
    _norm_within(out, ref["r"], "r")
    for got, name in zip(grads, ("dx", "dr", "dw", "dpost", "dgate")):
        _norm_within(got, ref[name], name)
    with torch.no_grad():
        z2, out2 = la.rmsnorm_residual(x, r, w, post, gate, 0.7)
    assert torch.equal(z2, z) and torch.equal(out2, out) and grads[4].dtype == torch.float32


def test_gates_of_other_types():
    """A float16 gate is exact in float32, a float64 one is rounded to it."""
    g = torch.Generator().manual_seed(1)
    x, gate = torch.randn(6, 128, generator=g).to(DEV, torch.bfloat16), torch.randn(6, 128, generator=g).to(DEV)
    for t in (torch.float16, torch.float64):
        other = gate.to(t).requires_grad_()
        _, out = la.rmsnorm_residual(x, None, None, None, other)
        _, want = la.rmsnorm_residual(x, None, None, None, other.detach().float())
        assert torch.equal(out, want)
        assert torch.autograd.grad(out, other, torch.ones_like(out))[0].dtype == t


# -- residual norm: without a norm behind the block an infinite x is like any other -------------------------------------

@pytest.mark.parametrize("d", [64, 65, 1000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinite_x_without_a_norm_has_a_finite_gradient(dtype, d):
    x, r, do = torch.ones(3, d, device=DEV, dtype=DT[dtype]), torch.zeros(3, d, device=DEV), torch.full((3, d), 2.0, device=DEV)
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    leaf = x.requires_grad_()
    z, out = la.rmsnorm_residual(leaf, r, torch.ones(d, device=DEV), None, None, 0.5)
    assert torch.isinf(out[1, 5]) and torch.isnan(out[2, 7])
    assert torch.equal(torch.autograd.grad(out, leaf, do)[0], torch.ones_like(x))


# -- captured passes ----------------------------------------------------------------------------------------------------

CALLS = {
    "recurrence": lambda x, c: la.gated_linear_recurrence(x, c)[0],
    "norm": lambda x, c: la.rmsnorm_residual(x, None, c)[0],
    "attention": lambda x, c: la.causal_attention(x, x, x),
}


def _leaf_and_constant(name):
    if name == "attention":
        return torch.randn(1, 1, 40, 64, device=DEV, requires_grad=True), None
    return torch.randn(1, 40, 64, device=DEV, requires_grad=True), -torch.ones(1, 40, 64, device=DEV) if name == "recurrence" else torch.ones(64, device=DEV)


@pytest.mark.parametrize("name", list(CALLS))
def test_a_leaf_behind_another_operation_is_seen(name):
    """The leaf's gradient would be added on the default stream, which cannot join the capture: the captured backward pass is refused."""
    leaf, c = _leaf_and_constant(name)
    free = torch.randn_like(leaf, requires_grad=True)
    alive = leaf * 2.0
    keep = torch.zeros(8, device=DEV)
    ones = torch.ones_like(leaf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep.add_(1)
        out = CALLS[name](leaf * 3.0 + free, c)
        with pytest.raises(RuntimeError, match="alive"):
            torch.autograd.grad(out, leaf, ones, retain_graph=True)
        with pytest.raises(RuntimeError, match="alive"):
            out.backward(ones, retain_graph=True)
        grad, = torch.autograd.grad(out, free, ones)  # does not touch the other leaf
    assert leaf.grad is None
    want, = torch.autograd.grad(CALLS[name]((leaf * 3.0).detach() + free, c), free, ones)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert bool((keep == i + 1).all()) and torch.equal(grad, want)
    del alive, out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad, = torch.autograd.grad(CALLS[name](leaf * 3.0 + free.detach(), c), leaf, ones)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, 3.0 * want)


# -- steps in place count as writes -------------------------------------------------------------------------------------

def _attention_step(kc, vc):
    q, k, v = (torch.randn(2, h, 64, device=DEV) for h in (4, 2, 2))
    la.causal_attention_step(q, k, v, kc, vc, torch.zeros(2, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("which", ["state", "k_cache", "v_cache"])
def test_what_a_step_overwrites_is_no_longer_what_was_saved(which):
    if which == "state":
        buf = torch.randn(3, 64, device=DEV)
        write = lambda: la.gated_linear_recurrence_step(torch.randn(3, 64, device=DEV), -torch.ones(3, 64, device=DEV), buf, inplace=True)
    else:
        buf, other = torch.randn(2, 2, 5, 64, device=DEV), torch.randn(2, 2, 5, 64, device=DEV)
        write = lambda: _attention_step(*((buf, other) if which == "k_cache" else (other, buf)))
    w = torch.ones_like(buf, requires_grad=True)
    saved = (w * buf[:]).sum()  # a view of it is saved
    before = buf._version
    write()
    assert buf._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    again = (w * buf).sum()
    again.backward()
    assert torch.equal(w.grad, buf)


def test_steps_in_inference_mode():
    with torch.inference_mode():
        state = torch.randn(3, 64, device=DEV)
        caches = [torch.randn(2, 2, 5, 64, device=DEV) for _ in "kv"]
        for _ in range(2):
            la.gated_linear_recurrence_step(state, -torch.ones_like(state), state, inplace=True)
            _attention_step(*caches)
    with torch.no_grad():  # tensors of inference mode have no version to count
        la.gated_linear_recurrence_step(torch.ones(3, 64, device=DEV), -torch.ones(3, 64, device=DEV), state, inplace=True)
        _attention_step(*caches)
    assert bool(torch.isfinite(state).all())
