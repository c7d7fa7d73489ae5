"""A pass that is captured while a graph of the same leaves from the default stream is alive is refused before anything is launched."""
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"


CALLS = {
    "recurrence": lambda x: la.gated_linear_recurrence(x, FIXED["g"])[0],
    "norm": lambda x: la.rmsnorm_residual(x, None, FIXED["w"])[0],
    "attention": lambda x: la.causal_attention(x, x, x),
}
FIXED = {}


@pytest.mark.parametrize("name", list(CALLS))
def test_refused_while_the_leaf_has_another_graph(name):
    FIXED.update(g=-torch.ones(1, 40, 64, device=DEV), w=torch.ones(64, device=DEV))
    leaf = torch.randn(*((1, 40, 64) if name == "recurrence" else (1, 1, 40, 64)), device=DEV, requires_grad=True)
    run = lambda: CALLS[name](leaf)
    alive = run()
    graph = torch.cuda.CUDAGraph()
    keep = torch.zeros(8, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        keep.add_(1)
        with pytest.raises(RuntimeError, match="alive"):
            run()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((keep == 1).all()) and bool(torch.isfinite(alive).all())
    del alive
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), torch.no_grad():
        want = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # the other graph is gone: the pass is captured
        out = run()
        grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool(torch.isfinite(grad).all())


@pytest.mark.parametrize("name", list(CALLS))
def test_warm_up_on_a_side_stream_may_be_alive(name):
    FIXED.update(g=-torch.ones(1, 40, 64, device=DEV), w=torch.ones(64, device=DEV))
    leaf = torch.randn(*((1, 40, 64) if name == "recurrence" else (1, 1, 40, 64)), device=DEV, requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = CALLS[name](leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = CALLS[name](leaf)
    for _ in range(3):
        with torch.no_grad():
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, alive)
