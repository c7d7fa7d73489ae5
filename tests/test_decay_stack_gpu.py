"""Layer norms, decay linear attention and causal attention as a hybrid stack runs them: three layers over packed documents with gradients
against float64, a prompt followed by decode tokens over pages, and decode steps of two streams as replayed graphs.

Tolerance of the stack: about sixteen operators in a row (products, norms, mixers and their gradients), each with float32 sums of at most
T + d + 64 terms, (T + d + 64) 2^-23 of its magnitude; residual additions and the norms of whole rows pass errors on without growth, the products of
this test by at most their weights' norm, below 4 in all, and a norm over a head's 16 columns with eps = 0.04 by at most 0.04 ** -0.5 = 5.
16 x (90 + 64 + 64) x 2^-23 x 4 x 5 = 8.4e-3 of the largest value."""
import pytest
import torch

import linearnexus_amd as la

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, H, HKV, HD, PAGE = 64, 4, 2, 16, 6
EPS = 0.04
TOL = 8.4e-3


def _weights():
    g = torch.Generator().manual_seed(21)
    n = lambda *s: torch.randn(*s, generator=g) * s[0] ** -0.5
    v = lambda *s: 1 + 0.2 * torch.randn(*s, generator=g)
    return dict(w1=v(D), b1=n(D), w2=v(D), b2=n(D), w3=v(D), qkv=n(D, 3 * H * HD), wg=n(D, H), wh=v(H, HD), bh=n(H, HD), wo=n(H * HD, D), wq=n(D, H * HD), wkv=n(D, 2 * HKV * HD),
                wo2=n(H * HD, D), qkv3=n(D, 3 * H * HD), decay=-0.05 * (1 + torch.rand(H, generator=g)), wo3=n(H * HD, D), wh3=v(HD))


def _heads(t, h):
    return t.view(*t.shape[:2], h, HD).transpose(1, 2)


def _mix(z, p, cu, qkv, g, weight, bias, states):
    """Decay attention and the norm of its heads."""
    q, k, v = (_heads(t, H) for t in (z @ p[qkv]).chunk(3, -1))
    o, state = la.decay_linear_attention(q, k, v, g, cu_seqlens=cu)
    states.append(state)
    return la.layer_norm(o.transpose(1, 2), weight, bias, EPS).flatten(2)


def _stack(x, p, cu, caches=None):
    states = []
    z = la.layer_norm(x, p["w1"], p["b1"])
    x = x + _mix(z, p, cu, "qkv", -torch.nn.functional.softplus(z @ p["wg"]).transpose(1, 2), p["wh"], p["bh"], states) @ p["wo"]
    z = la.layer_norm(x, p["w2"], p["b2"])
    k, v = (_heads(t, HKV) for t in (z @ p["wkv"]).chunk(2, -1))
    if caches is not None:
        caches.extend([k, v])
    x = x + la.causal_attention(_heads(z @ p["wq"], H), k, v, cu_seqlens=cu).transpose(1, 2).flatten(2) @ p["wo2"]
    z = la.layer_norm(x, p["w3"])
    x = x + _mix(z, p, cu, "qkv3", p["decay"], p["wh3"], None, states) @ p["wo3"]
    return la.layer_norm(x), states


def _plain(x, p, cu):
    """The same in elementary operations, one document at a time."""
    def norm(t, w=1.0, b=0.0, eps=1e-5):
        c = t - t.mean(-1, keepdim=True)
        return c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps) * w + b

    def mix(z, qkv, a, w, b):
        q, k, v = (z @ p[qkv]).view(-1, 3, H, HD).unbind(1)
        s, os = torch.zeros(H, HD, HD, dtype=z.dtype), []
        for t in range(z.shape[0]):
            s = a[t][:, None, None] * s + k[t][:, :, None] * v[t][:, None, :]
            os.append(HD ** -0.5 * (q[t][:, None] @ s)[:, 0])
        return norm(torch.stack(os), w, b, EPS).flatten(1), s

    zs, s1, s3 = [], [], []
    for lo, hi in zip(cu[:-1], cu[1:]):
        e = x[0, lo:hi]
        z = norm(e, p["w1"], p["b1"])
        m, s = mix(z, "qkv", torch.exp(-torch.nn.functional.softplus(z @ p["wg"])), p["wh"], p["bh"])
        s1.append(s)
        e = e + m @ p["wo"]
        z = norm(e, p["w2"], p["b2"])
        q, kv = (z @ p["wq"]).view(-1, H, HD), (z @ p["wkv"]).view(-1, 2, HKV, HD)
        k, v = (kv[:, i].repeat_interleave(H // HKV, 1) for i in (0, 1))
        s = torch.einsum("ihd,jhd->hij", q, k) * HD ** -0.5
        s = s.masked_fill(torch.ones(hi - lo, hi - lo, dtype=torch.bool).triu(1), float("-inf"))
        e = e + torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).flatten(1) @ p["wo2"]
        m, s = mix(norm(e, p["w3"]), "qkv3", torch.exp(p["decay"]).expand(hi - lo, H), p["wh3"], 0.0)
        s3.append(s)
        zs.append(norm(e + m @ p["wo3"]))
    return torch.cat(zs)[None], [torch.stack(s1), torch.stack(s3)]


def test_training_step_of_a_stack_on_packed_documents():
    cu = [0, 1, 34, 90]
    g = torch.Generator().manual_seed(3)
    x, cz = (torch.randn(1, 90, D, generator=g) for _ in range(2))
    cs = [torch.randn(3, H, HD, HD, generator=g) for _ in range(2)]
    names = sorted(_weights())
    got = {}
    for side, dev, dt, fn in (("ops", DEV, torch.float32, _stack), ("plain", "cpu", torch.float64, _plain)):
        leaves = [x.to(dev, dt).requires_grad_()] + [_weights()[n].to(dev, dt).requires_grad_() for n in names]
        z, states = fn(leaves[0], dict(zip(names, leaves[1:])), cu)
        loss = (z * cz.to(dev, dt)).sum() + sum((s * c.to(dev, dt)).sum() for s, c in zip(states, cs))
        got[side] = [t.detach().double().cpu() for t in (z, *states, *torch.autograd.grad(loss, leaves))]
    for what, a, b in zip(("z", "state 1", "state 3", "dx", *names), got["ops"], got["plain"]):
        assert float((a - b).abs().max()) < TOL * float(b.abs().max()), what


class _Decoder:
    """One token a call through all layers, all state in place; the pages of the sequences lie in between each other."""

    def __init__(self, p, batch, places):
        self.p = p
        self.x = torch.zeros(batch, D, device=DEV)
        self.states = [torch.zeros(batch, H, HD, HD, device=DEV) for _ in range(2)]
        width = -(-places // PAGE)
        self.table = torch.randperm(batch * width, generator=torch.Generator().manual_seed(1)).view(batch, width).to(DEV, torch.int32)
        self.k, self.v = (torch.zeros(batch * width, HKV, PAGE, HD, device=DEV) for _ in range(2))
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)

    def prompt(self, states, k, v):
        for own, s in zip(self.states, states):
            own.copy_(s)
        n = k.shape[2]
        for b in range(k.shape[0]):
            for j in range(n):
                page = int(self.table[b, j // PAGE])
                self.k[page, :, j % PAGE], self.v[page, :, j % PAGE] = k[b, :, j], v[b, :, j]
        self.lengths.fill_(n)

    def _mix(self, z, i, qkv, g, weight, bias):
        q, k, v = (t.view(-1, H, HD) for t in (z @ self.p[qkv]).chunk(3, -1))
        o, _ = la.decay_linear_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), g, self.states[i], inplace=True)
        return la.layer_norm(o, weight, bias, EPS).flatten(1)

    def token(self):
        p, x = self.p, self.x
        z = la.layer_norm(x, p["w1"], p["b1"])
        x = x + self._mix(z, 0, "qkv", -torch.nn.functional.softplus(z @ p["wg"]), p["wh"], p["bh"]) @ p["wo"]
        z = la.layer_norm(x, p["w2"], p["b2"])
        kv = (z @ p["wkv"]).view(-1, 2, HKV, HD)
        o = la.causal_attention_step_paged((z @ p["wq"]).view(-1, H, HD), kv[:, 0], kv[:, 1], self.k, self.v, self.table, self.lengths)
        self.lengths.add_(1)
        x = x + o.flatten(1) @ p["wo2"]
        z = la.layer_norm(x, p["w3"])
        return la.layer_norm(x + self._mix(z, 1, "qkv3", p["decay"], p["wh3"], None) @ p["wo3"])


def test_decode_tokens_continue_a_prompt():
    p = {n: t.to(DEV) for n, t in _weights().items()}
    x = torch.randn(2, 60, D, generator=torch.Generator().manual_seed(5)).to(DEV)
    whole = _stack(x, p, None)[0]
    dec, cache = _Decoder(p, 2, 64), []
    _, states = _stack(x[:, :50], p, None, cache)
    dec.prompt(states, *cache)
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
        for s in d.states:
            s.zero_()
        d.lengths.zero_()
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_segmented_prompts_on_two_streams(dtype):
    """Long rows are walked in segments through workspaces: calls on two streams, a side stream's inputs used right after, and replays all agree."""
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(1, 2, 2100, 32, generator=g).to(DEV, dtype) for _ in range(3))
    a = -torch.rand(1, 2, 2100, generator=g).to(DEV) * 0.1
    go = torch.randn(1, 2, 2100, 32, generator=g).to(DEV, dtype)

    def call():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, a)]
        o, s = la.decay_linear_attention(*leaves)
        return [o.detach(), s.detach(), *torch.autograd.grad((o, s), leaves, (go, torch.ones_like(s)))]

    want = call()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for turn in range(4):
        with torch.cuda.stream(streams[turn % 2]):
            got.append(call())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        graph.replay()
        got.append([t.clone() for t in out])
        torch.cuda.synchronize()
    for run in got:
        for x, y in zip(run, want):
            assert torch.equal(x, y)
