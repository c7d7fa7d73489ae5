"""The residual norms, the gated linear recurrence and causal attention as a hybrid stack runs them: two layers over packed documents
with gradients against float64, a prompt followed by decode tokens, and the decode step of two streams as replayed graphs.

Tolerance of the stack: about twelve operators in a row (products, norms, recurrence, attention and their gradients), each with float32
sums of at most T + d + 64 terms, (T + d + 64) 2^-23 of its magnitude; norms and residual additions pass errors on without growth, the
products of this test by at most their weights' norm, below 4 in all.  12 x (90 + 64 + 64) x 2^-23 x 4 = 1.2e-3 of the largest value."""
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, H, HKV, HD = 64, 4, 2, 16
TOL = 1.2e-3


def _weights(dtype=torch.float32):
    g = torch.Generator().manual_seed(11)
    n = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).to(dtype)
    v = lambda: (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)
    return dict(w1=v(), w2=v(), w3=v(), p1=v(), p2=v(), s1=0.5 * v(), wx=n(D, D), wg=n(D, D), wo=n(D, D), gate=n(D, D), wq=n(D, H * HD), wkv=n(D, 2 * HKV * HD),
                wo2=n(H * HD, D))


def _heads(t, h):
    return t.view(*t.shape[:2], h, HD).transpose(1, 2)


def _stack(x, p, cu):
    """The layers through the library's ops."""
    z, r = la.rmsnorm_residual(x, None, p["w1"])
    y, state = la.gated_linear_recurrence(z @ p["wx"], -torch.nn.functional.softplus(z @ p["wg"]), cu_seqlens=cu)
    z, r = la.rmsnorm_residual(y @ p["wo"], r, p["w2"], p["p1"], z @ p["gate"], p["s1"])
    kv = z @ p["wkv"]
    o = la.causal_attention(_heads(z @ p["wq"], H), _heads(kv[..., : HKV * HD], HKV), _heads(kv[..., HKV * HD :], HKV), cu_seqlens=cu)
    z, r = la.rmsnorm_residual(o.transpose(1, 2).reshape(*x.shape[:2], H * HD) @ p["wo2"], r, p["w3"], p["p2"], None, 0.7)
    return z, r, state


def _plain(x, p, cu):
    """The same in elementary operations, one document at a time."""
    norm = lambda t, w: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5) * w
    zs, rs, states = [], [], []
    for lo, hi in zip(cu[:-1], cu[1:]):
        e = x[0, lo:hi]
        z, r = norm(e, p["w1"]), e
        u, a = z @ p["wx"], torch.exp(-torch.nn.functional.softplus(z @ p["wg"]))
        h, ys = torch.zeros_like(u[0]), []
        for t in range(hi - lo):
            h = a[t] * h + u[t]
            ys.append(h)
        states.append(h)
        r = r + p["s1"] * torch.sigmoid(z @ p["gate"]) * norm(torch.stack(ys) @ p["wo"], p["p1"])
        z = norm(r, p["w2"])
        q, kv = (z @ p["wq"]).view(-1, H, HD), (z @ p["wkv"]).view(-1, 2, HKV, HD)
        k, v = (kv[:, i].repeat_interleave(H // HKV, 1) for i in (0, 1))
        s = torch.einsum("ihd,jhd->hij", q, k) * HD ** -0.5
        s = s.masked_fill(torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        o = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(hi - lo, H * HD)
        r = r + 0.7 * norm(o @ p["wo2"], p["p2"])
        zs.append(norm(r, p["w3"]))
        rs.append(r)
    return torch.cat(zs)[None], torch.cat(rs)[None], torch.stack(states)


def test_training_step_of_a_stack_on_packed_documents():
    cu = [0, 1, 34, 90]
    g = torch.Generator().manual_seed(3)
    x, cz, cr, cs = (torch.randn(*s, generator=g) for s in ((1, 90, D), (1, 90, D), (1, 90, D), (3, D)))
    names = sorted(_weights())
    got = {}
    for side, dev, dt, fn in (("ops", DEV, torch.float32, _stack), ("plain", "cpu", torch.float64, _plain)):
        leaves = [x.to(dev, dt).requires_grad_()] + [_weights()[n].to(dev, dt).requires_grad_() for n in names]
        z, r, s = fn(leaves[0], dict(zip(names, leaves[1:])), cu)
        loss = (z * cz.to(dev, dt)).sum() + (r * cr.to(dev, dt)).sum() + (s * cs.to(dev, dt)).sum()
        got[side] = [t.detach().double().cpu() for t in (z, r, s, *torch.autograd.grad(loss, leaves))]
    for what, a, b in zip(("z", "r", "state", "dx", *names), got["ops"], got["plain"]):
        assert float((a - b).abs().max()) < TOL * float(b.abs().max()), what


class _Decoder:
    """One token a call through both layers, all state in place."""

    def __init__(self, p, batch, places):
        self.p = p
        self.x = torch.zeros(batch, D, device=DEV)
        self.state = torch.zeros(batch, D, device=DEV)
        self.k, self.v = (torch.zeros(batch, HKV, places, HD, device=DEV) for _ in range(2))
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)

    def token(self):
        p, b = self.p, self.x.shape[0]
        z, r = la.rmsnorm_residual(self.x, None, p["w1"])
        y, _ = la.gated_linear_recurrence_step(z @ p["wx"], -torch.nn.functional.softplus(z @ p["wg"]), self.state, inplace=True)
        z, r = la.rmsnorm_residual(y @ p["wo"], r, p["w2"], p["p1"], z @ p["gate"], p["s1"])
        kv = (z @ p["wkv"]).view(b, 2, HKV, HD)
        o = la.causal_attention_step((z @ p["wq"]).view(b, H, HD), kv[:, 0], kv[:, 1], self.k, self.v, self.lengths)
        self.lengths.add_(1)
        return la.rmsnorm_residual(o.reshape(b, H * HD) @ p["wo2"], r, p["w3"], p["p2"], None, 0.7)[0]


def test_decode_tokens_continue_a_prompt():
    p = {n: t.to(DEV) for n, t in _weights().items()}
    x = torch.randn(2, 60, D, generator=torch.Generator().manual_seed(5)).to(DEV)
    whole = _stack(x, p, None)[0]
    dec = _Decoder(p, 2, 64)
    # the prompt through the whole-sequence ops, its keys and values into the cache
    z, r = la.rmsnorm_residual(x[:, :50], None, p["w1"])
    y, state = la.gated_linear_recurrence(z @ p["wx"], -torch.nn.functional.softplus(z @ p["wg"]))
    z, _ = la.rmsnorm_residual(y @ p["wo"], r, p["w2"], p["p1"], z @ p["gate"], p["s1"])
    kv = z @ p["wkv"]
    dec.state.copy_(state)
    dec.k[:, :, :50], dec.v[:, :, :50] = _heads(kv[..., : HKV * HD], HKV), _heads(kv[..., HKV * HD :], HKV)
    dec.lengths.fill_(50)
    for t in range(50, 60):
        dec.x.copy_(x[:, t])
        out = dec.token()
        assert float((out - whole[:, t]).abs().max()) < TOL * float(whole.abs().max())


def test_two_decoders_as_graphs_side_by_side():
    """Two captured decode steps share nothing: replayed in turn and on two streams they give what eager calls give."""
    p = {n: t.to(DEV) for n, t in _weights().items()}
    g = torch.Generator().manual_seed(6)
    xs = [torch.randn(b, 12, D, generator=g).to(DEV) for b in (1, 3)]
    want = []
    for x in xs:
        dec, outs = _Decoder(p, x.shape[0], 400), []
        for t in range(12):
            dec.x.copy_(x[:, t])
            outs.append(dec.token())
        want.append(torch.stack(outs, 1))
    decs = [_Decoder(p, x.shape[0], 400) for x in xs]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in decs:
            d.token()
    torch.cuda.current_stream().wait_stream(side)
    for d in decs:
        d.state.zero_(), d.lengths.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(d.token())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for t in range(12):
        for i, (d, x) in enumerate(zip(decs, xs)):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                d.x.copy_(x[:, t])
                graphs[i].replay()
                got[i].append(outs[i].clone())
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(torch.stack(a, 1), b)
