"""More operators of a hybrid layer stack -- linear attention with a decay for each head, layer norms, and one decode token's
attention over a paged cache -- as cases that can be timed and compared.

``listed()`` gives the fixed cases and ``draw(rng)`` one more of the same ranges; ``prepare`` makes what a program holds
before the call, ``run`` is one pass, ``work`` what that pass cannot do without, and ``exact`` the pass's outputs from the
operators' definitions in 64 bits.  With ``own`` false a pass is the plain form in elementary torch operations in float32 (sums of
log-decays in float64), rounded once at the end; with ``own`` true it is the library's operator as a user calls it.

Kinds of case:

``decay``       ``S_t = e^{g_t} S_{t-1} + k_t^T v_t``, ``o_t = scale q_t S_t`` over whole sequences, dense or packed, ``g`` for each token or one
                constant for each head; with ``grad`` the backward pass too.
``decay_step``  one decode token of it, the new state beside the old one.
``norm``        ``y = (x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, the weights ``[d]`` or ``[heads, d]``; with
                ``grad`` the backward pass.
``paged``       one decode token of causal attention with grouped heads against keys and values in pages: the token is appended, then attends.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
EPS = 1e-5


def _decay(B, H, T, dk, dv, dtype, *, g, nseq=0, grad, state, token_first, name=None):
    c = {"kind": "decay", "B": B, "H": H, "T": T, "dk": dk, "dv": dv, "dtype": dtype, "g": g, "nseq": nseq, "grad": grad, "state": state, "token_first": token_first}
    return c if name is None else {"name": name, **c}


def _decay_step(B, H, dk, dv, dtype, name=None):
    c = {"kind": "decay_step", "B": B, "H": H, "dk": dk, "dv": dv, "dtype": dtype}
    return c if name is None else {"name": name, **c}


def _norm(rows, heads, d, dtype, *, bias, grad, name=None):
    c = {"kind": "norm", "rows": rows, "heads": heads, "d": d, "dtype": dtype, "bias": bias, "grad": grad}
    return c if name is None else {"name": name, **c}


def _paged(B, H, Hkv, S, page, d, dtype, *, token_first, name=None):
    c = {"kind": "paged", "B": B, "H": H, "Hkv": Hkv, "S": S, "page": page, "d": d, "dtype": dtype, "token_first": token_first}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # the mixer of a training step at the repository's headline batch (8 x 4096 tokens, 16 heads of 128), tensors as the projections leave them
        _decay(8, 16, 4096, 128, 128, "bf16", g="token", grad=True, state=False, token_first=True, name="decay_train"),
        # one very long prompt being prefilled at an odd length, fixed decays for each head, the state kept for decoding
        _decay(1, 16, 65000, 128, 128, "bf16", g="head", grad=False, state=True, token_first=True, name="decay_prompt_t65000"),
        # a small model in float32 on packed documents of ragged length, their states handed on
        _decay(1, 6, 2503, 64, 96, "f32", g="token", nseq=7, grad=True, state=True, token_first=False, name="decay_packed_f32"),
        # one decode token of a server's batch (the repository's decode configuration, 32 heads of 128)
        _decay_step(256, 32, 128, 128, "bf16", name="decay_step_b256"),
        # one user's decode token: latency
        _decay_step(1, 16, 128, 128, "bf16", name="decay_step_b1"),
        # the norm before a block in the same training step
        _norm(32768, 1, 2048, "bf16", bias=True, grad=True, name="norm_train"),
        # the norm of each head behind the mixer in that step, a weight for every head
        _norm(32768, 16, 128, "bf16", bias=True, grad=True, name="norm_heads"),
        # an odd number of rows of an odd width in float32, no bias
        _norm(2007, 1, 1001, "f32", bias=False, grad=True, name="norm_ragged_f32"),
        # one decode token of a small batch: latency
        _norm(27, 1, 4096, "bf16", bias=True, grad=False, name="norm_token_b27"),
        # one decode token of a server's batch over long paged caches
        _paged(32, 32, 8, 8192, 64, 128, "bf16", token_first=True, name="paged_b32"),
        # one user's decode token, a short odd cache in small pages: latency
        _paged(1, 16, 4, 1000, 16, 128, "bf16", token_first=False, name="paged_b1"),
        # a small float32 model's batch, pages of an odd size
        _paged(7, 6, 2, 3001, 48, 64, "f32", token_first=False, name="paged_f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["decay", "decay", "decay", "decay_step", "norm", "norm", "paged", "paged"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    grad = rng.random() < 0.5
    if kind == "decay":
        dk, dv = rng.choice([64, 128, 128, 80, 256]), rng.choice([64, 128, 128, 96, 256])
        H, T = rng.randint(1, 24), _log(rng, 1, 65536)
        most = (1 << 26) if dtype == "bf16" else (1 << 23)  # elements of the wider tensors
        T = max(1, min(T, most // (H * max(dk, dv))))
        B = max(1, min(_log(rng, 1, 16), most // (H * T * max(dk, dv))))
        nseq = rng.randint(1, min(T, 24)) if rng.random() < 0.4 else 0
        return _decay(1 if nseq else B, H, T, dk, dv, dtype, g=rng.choice(["token", "token", "head"]), nseq=nseq, grad=grad, state=rng.random() < 0.5,
                      token_first=rng.random() < 0.5)
    if kind == "decay_step":
        return _decay_step(_log(rng, 1, 256), _log(rng, 1, 32), rng.choice([64, 128, 80]), rng.choice([64, 128, 96]), dtype)
    if kind == "norm":
        heads = rng.choice([1, 1, rng.randint(2, 16)])
        d = _log(rng, 64, 8192) if heads == 1 else _log(rng, 32, 512)
        rows = max(1, min(_log(rng, 1, 32768), (1 << 25) // (d * heads)))
        return _norm(rows, heads, d, dtype, bias=rng.random() < 0.6, grad=grad)
    Hkv = rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 128, 128, 80, 40])
    S = _log(rng, 1, 8192)
    B = max(1, min(_log(rng, 1, 64), (1 << 24) // (Hkv * S * max(1, d // 16))))
    return _paged(B, Hkv * rng.choice([1, 2, 3, 4, 8]), Hkv, S, rng.choice([1, 8, 16, 16, 24, 64, 128, 256]), d, dtype, token_first=rng.random() < 0.5)


def _lengths(case):
    """Lengths of the packed sequences, at least one token each, summing to T: the same for every seed of a case, as `work` needs them."""
    r = random.Random(case["nseq"] * 1000003 + case["T"])
    cuts = sorted(r.sample(range(1, case["T"]), case["nseq"] - 1))
    return [b - a for a, b in zip([0, *cuts], [*cuts, case["T"]])]


def _fills(case):
    """Tokens that each sequence of a decode batch already holds: ragged, between half of the places and all but the last."""
    r = random.Random(case["B"] * 1000003 + case["S"])
    return [r.randint((case["S"] - 1) // 2, case["S"] - 1) for _ in range(case["B"])]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def n(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std).to(dtype)

    def rates(H):
        # decays of a trained gate: time constants from one token to a thousand, spread over the heads
        return torch.exp(torch.rand(H, generator=gen, device=DEVICE) * math.log(1000.0)).reciprocal()

    s = {"case": case}
    if case["kind"] == "decay":
        B, H, T, dk, dv = (case[x] for x in ("B", "H", "T", "dk", "dv"))

        def heads(d):
            return n(B, T, H, d).transpose(1, 2) if case["token_first"] else n(B, H, T, d)

        s.update(q=heads(dk), k=heads(dk), v=heads(dv), state=None, cu=None, lens=None)
        if case["g"] == "head":
            s["g"] = -rates(H)
        else:
            z = torch.nn.functional.softplus(n(B, T, H, dtype=torch.float32) + 0.5)
            s["g"] = (-rates(H) * z).transpose(1, 2)
            if not case["token_first"]:
                s["g"] = s["g"].contiguous()
        rows = B
        if case["nseq"]:
            s["lens"], rows = _lengths(case), case["nseq"]
            s["cu"] = torch.tensor([0, *torch.tensor(s["lens"]).cumsum(0).tolist()], dtype=torch.int32, device=DEVICE)
        if case["state"]:
            s["state"] = n(rows, H, dk, dv, dtype=torch.float32)
        if case["grad"]:
            s.update(do=heads(dv), ds=n(rows, H, dk, dv, std=0.1, dtype=torch.float32))
    elif case["kind"] == "decay_step":
        B, H, dk, dv = (case[x] for x in ("B", "H", "dk", "dv"))
        s.update(q=n(B, H, dk), k=n(B, H, dk), v=n(B, H, dv), state=n(B, H, dk, dv, dtype=torch.float32))
        s["g"] = -rates(H) * torch.nn.functional.softplus(n(B, H, dtype=torch.float32) + 0.5)
    elif case["kind"] == "norm":
        rows, heads, d = case["rows"], case["heads"], case["d"]
        shape = (rows, heads, d) if heads > 1 else (rows, d)
        s.update(x=n(*shape, std=2.0) + n(*shape[:-1], 1), w=1 + n(*shape[1:], std=0.2, dtype=torch.float32), b=None)
        if case["bias"]:
            s["b"] = n(*shape[1:], std=0.2, dtype=torch.float32)
        if case["grad"]:
            s["dy"] = n(*shape)
    else:
        B, H, Hkv, S, page, d = (case[x] for x in ("B", "H", "Hkv", "S", "page", "d"))
        fills, per = _fills(case), -(-S // page)
        used = [f // page + 1 for f in fills]
        P = sum(used) + 3  # a pool with pages to spare, handed out in no order
        ids = torch.randperm(P, generator=gen, device=DEVICE).to(torch.int32)
        table = torch.full((B, per), -1, dtype=torch.int32, device=DEVICE)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = ids[at : at + u]
            at += u

        def pages():
            return n(P, page, Hkv, d).transpose(1, 2) if case["token_first"] else n(P, Hkv, page, d)

        s.update(q=n(B, H, d, std=1.5), k=n(B, Hkv, d), v=n(B, Hkv, d), kp=pages(), vp=pages(), table=table, fill=torch.tensor(fills, dtype=torch.int32, device=DEVICE))
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------

CHUNK = 64


def _decay_rows(q, k, v, g, s0, do, ds):
    """Rows of one length, ``[B,H,T,.]`` in float32 and g in float64, chunk by chunk: outputs, last state and, with do, the gradients."""
    B, H, T, dk = q.shape
    dv, n, scale = v.shape[-1], -(-T // CHUNK), dk ** -0.5

    def cut(t):
        t = torch.nn.functional.pad(t, (0, 0, 0, n * CHUNK - T))
        return t.reshape(B, H, n, CHUNK, t.shape[-1])

    q, k, v, g = cut(q * scale), cut(k), cut(v), cut(g[..., None])[..., 0]
    G = g.cumsum(-1)
    total = G[..., -1:]
    keep = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    pair = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill_(~keep, float("-inf"))).float()
    into, out_of, whole = torch.exp(G).float()[..., None], torch.exp(total - G).float()[..., None], torch.exp(total).float()[..., None]
    A = torch.matmul(q, k.transpose(-1, -2).contiguous()) * pair
    o = torch.matmul(A, v)
    S = torch.zeros(B, H, dk, dv, device=q.device) if s0 is None else s0.float()
    before = []
    for c in range(n):
        before.append(S)
        o[:, :, c] += torch.matmul(q[:, :, c] * into[:, :, c], S)
        S = whole[:, :, c] * S + torch.matmul((k[:, :, c] * out_of[:, :, c]).transpose(-1, -2), v[:, :, c])

    def back(t):
        return t.reshape(B, H, n * CHUNK, t.shape[-1])[:, :, :T]

    res = {"o": back(o), "state": S}
    if do is None:
        return res
    do = cut(do)
    dv_ = torch.matmul(A.transpose(-1, -2), do)
    dA = torch.matmul(do, v.transpose(-1, -2).contiguous()) * pair
    dq, dk_ = torch.matmul(dA, k), torch.matmul(dA.transpose(-1, -2), q)
    del A, dA, pair
    dS = ds
    dG = torch.zeros_like(G)
    for c in range(n - 1, -1, -1):
        dG[:, :, c, -1] += (dS * whole[:, :, c] * before[c]).double().sum((-1, -2))
        y = torch.matmul(v[:, :, c] * out_of[:, :, c], dS.transpose(-1, -2).contiguous())
        x = torch.matmul(do[:, :, c] * into[:, :, c], before[c].transpose(-1, -2).contiguous())
        # a token's decay acts on what came before it: the terms that its outputs and the later ones take from the state, and what the
        # chunk's earlier keys hand on
        dG[:, :, c] += (x * q[:, :, c]).double().sum(-1)
        handed = (y * k[:, :, c]).double().sum(-1)
        dG[:, :, c, -1] += handed.sum(-1)
        dG[:, :, c] -= handed
        # pairs within the chunk
        dG[:, :, c] += (dq[:, :, c] * q[:, :, c]).double().sum(-1) - (dk_[:, :, c] * k[:, :, c]).double().sum(-1)
        dk_[:, :, c] += y
        dq[:, :, c] += x
        dv_[:, :, c] += torch.matmul(k[:, :, c] * out_of[:, :, c], dS)
        dS = whole[:, :, c] * dS + torch.matmul((q[:, :, c] * into[:, :, c]).transpose(-1, -2), do[:, :, c])
    dg = dG.flip(-1).cumsum(-1).flip(-1)
    res.update(dq=back(dq) * scale, dk=back(dk_), dv=back(dv_), dg=back(dg[..., None])[..., 0], dstate=dS)
    return res


def _decay_plain(s):
    case, grad = s["case"], "do" in s
    B, H, T = case["B"], case["H"], case["T"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    g = s["g"].double()
    if case["g"] == "head":
        g = g[None, :, None].expand(B, H, T)
    if s["lens"] is None:
        parts = [_decay_rows(q, k, v, g, s["state"], s["do"].float() if grad else None, s.get("ds"))]
    else:
        parts, lo = [], 0
        for i, n in enumerate(s["lens"]):
            w = slice(lo, lo + n)
            lo += n
            parts.append(_decay_rows(q[:, :, w], k[:, :, w], v[:, :, w], g[:, :, w], None if s["state"] is None else s["state"][i : i + 1],
                                     s["do"][:, :, w].float() if grad else None, s["ds"][i : i + 1] if grad else None))
    dt = s["q"].dtype

    def rows(name):
        return torch.cat([p[name] for p in parts], 2) if len(parts) > 1 else parts[0][name]

    def states(name):
        return torch.cat([p[name] for p in parts], 0) if len(parts) > 1 else parts[0][name]

    out = {"o": rows("o").to(dt), "state": states("state")}
    if grad:
        dg = rows("dg")
        out.update(dq=rows("dq").to(dt), dk=rows("dk").to(dt), dv=rows("dv").to(dt), dg=(dg.sum((0, 2)) if case["g"] == "head" else dg).float())
        if s["state"] is not None:
            out["dstate"] = states("dstate")
    return out


def _decay_own(s):
    import linearnexus_amd as la
    if "do" not in s:
        o, state = la.decay_linear_attention(s["q"], s["k"], s["v"], s["g"], None, s["state"], cu_seqlens=s["cu"])
        return {"o": o, "state": state}
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "state") if s[n] is not None]
    o, state = la.decay_linear_attention(*leaves[:4], None, leaves[4] if len(leaves) > 4 else None, cu_seqlens=s["cu"])
    grads = torch.autograd.grad([o, state], leaves, [s["do"], s["ds"]])
    return {"o": o.detach(), "state": state.detach(), **dict(zip(("dq", "dk", "dv", "dg", "dstate"), grads))}


def _decay_step_run(s):
    if own:
        import linearnexus_amd as la
        o, state = la.decay_linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"])
        return {"o": o, "state": state}
    k, v = s["k"].float(), s["v"].float()
    S = torch.exp(s["g"])[..., None, None] * s["state"] + k[..., :, None] * v[..., None, :]
    o = torch.matmul(s["q"].float()[..., None, :] * s["case"]["dk"] ** -0.5, S)[..., 0, :]
    return {"o": o.to(s["q"].dtype), "state": S}


def _norm_run(s):
    if own:
        import linearnexus_amd as la
        if "dy" not in s:
            return {"y": la.layer_norm(s["x"], s["w"], s["b"], EPS)}
        leaves = [s[n].detach().requires_grad_() for n in ("x", "w", "b") if s[n] is not None]
        y = la.layer_norm(leaves[0], leaves[1], leaves[2] if len(leaves) > 2 else None, EPS)
        return {"y": y.detach(), **dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, s["dy"])))}
    x, w = s["x"].float(), s["w"]
    x = x - x.mean(-1, keepdim=True)
    rho = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * rho
    out = {"y": (xh * w if s["b"] is None else xh * w + s["b"]).to(s["x"].dtype)}
    if "dy" in s:
        dy = s["dy"].float()
        u = dy * w
        out["dx"] = (rho * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))).to(s["x"].dtype)
        out["dw"] = (dy * xh).sum(0)
        if s["b"] is not None:
            out["db"] = dy.sum(0)
    return out


def _paged_run(s):
    case = s["case"]
    B, H, Hkv, S, page, d = (case[x] for x in ("B", "H", "Hkv", "S", "page", "d"))
    if own:
        import linearnexus_amd as la
        o = la.causal_attention_step_paged(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["fill"])
        return {"o": o, "k": s["kp"], "v": s["vp"]}
    at = s["fill"].long()
    row = torch.arange(B, device=at.device)
    where = s["table"][row, at // page].long()
    s["kp"][where, :, at % page] = s["k"]
    s["vp"][where, :, at % page] = s["v"]
    ids = s["table"].clamp(min=0).long()

    def cache(t):  # [B, Hkv, places, d]
        return t[ids].float().transpose(1, 2).reshape(B, Hkv, -1, d)

    q = s["q"].float().view(B, Hkv, H // Hkv, d) * d ** -0.5
    sc = torch.matmul(q, cache(s["kp"]).transpose(2, 3).contiguous())
    hide = (torch.arange(sc.shape[-1], device=q.device) > at[:, None])[:, None, None]
    sc = sc.masked_fill_(hide, float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p / p.sum(-1, keepdim=True), cache(s["vp"]))
    return {"o": o.reshape(B, H, d).to(s["q"].dtype), "k": s["kp"], "v": s["vp"]}


def run(state):
    kind = state["case"]["kind"]
    if kind == "decay":
        return _decay_own(state) if own else _decay_plain(state)
    if kind == "decay_step":
        return _decay_step_run(state)
    if kind == "norm":
        return _norm_run(state)
    return _paged_run(state)


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "decay":
        B, H, T, dk, dv = (case[x] for x in ("B", "H", "T", "dk", "dv"))
        rows = case["nseq"] or B
        tokens = B * H * T
        gates = 4 * (H if case["g"] == "head" else tokens)
        states = rows * H * dk * dv * 4
        moved = tokens * 2 * (dk + dv) * e + gates + states * (1 + case["state"])  # q, k, v, o; g; the states
        flops = tokens * 4 * dk * dv
        if case["grad"]:
            moved += tokens * 2 * (dk + dv) * e + gates + states * (1 + case["state"])  # do, dq, dk, dv; dg; the states' gradients
            flops = tokens * 14 * dk * dv
        return {"bytes": moved, "flops": flops}
    if kind == "decay_step":
        B, H, dk, dv = (case[x] for x in ("B", "H", "dk", "dv"))
        return {"bytes": B * H * (8 * dk * dv + 2 * (dk + dv) * e + 4), "flops": B * H * dk * dv * 5}
    if kind == "norm":
        n, width = case["rows"] * case["heads"] * case["d"], case["heads"] * case["d"]
        vectors = 4 * width * (1 + case["bias"])
        return {"bytes": n * e * 2 + vectors + (n * e * 2 + vectors if case["grad"] else 0), "flops": n * (24 if case["grad"] else 8)}
    B, H, Hkv, d = (case[x] for x in ("B", "H", "Hkv", "d"))
    keys = sum(f + 1 for f in _fills(case))
    pages = sum(f // case["page"] + 1 for f in _fills(case))
    return {"bytes": keys * Hkv * d * e * 2 + B * (2 * H + 4 * Hkv) * d * e + 4 * pages, "flops": keys * H * d * 4}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "decay":
        return _decay_exact(case, s)
    if kind == "decay_step":
        S = s["state"].double() * s["g"].double().exp()[..., None, None]
        S += s["k"].double().unsqueeze(-1) * s["v"].double().unsqueeze(-2)
        return {"o": (s["q"].double().unsqueeze(-1) * S).sum(-2) / math.sqrt(case["dk"]), "state": S}
    if kind == "norm":
        leaf = {n: s[n].double().requires_grad_() for n in ("x", "w", "b") if s[n] is not None}
        x = leaf["x"]
        y = (x - x.mean(-1, True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + EPS) * leaf["w"] + leaf.get("b", 0.0)
        out = {"y": y.detach()}
        if case["grad"]:
            out.update(zip(("dx", "dw", "db"), torch.autograd.grad(y, list(leaf.values()), s["dy"].double())))
        return out
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group, page = case["H"] // case["Hkv"], case["page"]
    for b, fill in enumerate(s["fill"].tolist()):
        used = s["table"][b, : fill // page + 1].tolist()
        kept = []
        for t, new in ((s["kp"], s["k"]), (s["vp"], s["v"])):
            whole = torch.cat([t[i] for i in used], 1).double()[:, : fill + 1]  # [Hkv, fill + 1, d]
            whole[:, fill] = new[b].double()
            kept.append(whole)
        for h in range(case["H"]):
            weight = torch.softmax(kept[0][h // group] @ s["q"][b, h].double() / math.sqrt(case["d"]), 0)
            o[b, h] = weight @ kept[1][h // group]
    return {"o": o, "k": None, "v": None}


BLOCK = 1024


def _decay_exact(case, s):
    """One sequence at a time, its heads in groups: the pairs of a block as a whole matrix, the state between blocks; gradients by automatic differentiation."""
    B, H, T, dk, dv, grad = (case[x] for x in ("B", "H", "T", "dk", "dv", "grad"))
    if B * H * T * (BLOCK + dk + dv) * (4.0 if grad else 1.0) * 1e-10 * 2 > 20 or B * H * T * max(dk, dv) > 1 << 27:
        return None
    if s["lens"]:
        ends = [sum(s["lens"][: i + 1]) for i in range(case["nseq"])]
        spans = [(0, lo, hi, i) for i, (lo, hi) in enumerate(zip([0, *ends], ends))]
    else:
        spans = [(b, 0, T, b) for b in range(B)]
    out = {"o": torch.zeros(B, H, T, dv, dtype=torch.float64, device=DEVICE), "state": torch.zeros(len(spans), H, dk, dv, dtype=torch.float64, device=DEVICE)}
    if grad:
        for name, like in (("dq", dk), ("dk", dk), ("dv", dv)):
            out[name] = torch.zeros(B, H, T, like, dtype=torch.float64, device=DEVICE)
        out["dg"] = torch.zeros((H,) if case["g"] == "head" else (B, H, T), dtype=torch.float64, device=DEVICE)
        if case["state"]:
            out["dstate"] = torch.zeros_like(out["state"])
    for b, lo, hi, i in spans:
        for h in range(0, H, 4):
            hs = slice(h, min(h + 4, H))
            q, k, v = (s[n][b, hs, lo:hi].double().requires_grad_(grad) for n in ("q", "k", "v"))
            g = (s["g"][hs] if case["g"] == "head" else s["g"][b, hs, lo:hi]).double().requires_grad_(grad)
            s0 = (torch.zeros(q.shape[0], dk, dv, dtype=torch.float64, device=DEVICE) if s["state"] is None else s["state"][i, hs].double()).requires_grad_(grad)
            steps = g[:, None].expand(-1, hi - lo) if case["g"] == "head" else g
            S, os = s0, []
            for t in range(0, hi - lo, BLOCK):
                w = slice(t, min(t + BLOCK, hi - lo))
                c = steps[:, w].cumsum(1)
                hide = torch.ones(c.shape[1], c.shape[1], dtype=torch.bool, device=DEVICE).triu(1)
                m = torch.exp((c.unsqueeze(2) - c.unsqueeze(1)).masked_fill(hide, -math.inf))
                rows = torch.bmm(torch.bmm(q[:, w], k[:, w].mT) * m, v[:, w]) + torch.bmm(q[:, w], S) * c.exp().unsqueeze(2)
                os.append(rows / math.sqrt(dk))
                last = c[:, -1:]
                S = S * last.exp().unsqueeze(2) + torch.bmm(k[:, w].mT, v[:, w] * (last - c).exp().unsqueeze(2))
            o = torch.cat(os, 1)
            out["o"][b, hs, lo:hi], out["state"][i, hs] = o.detach(), S.detach()
            if not grad:
                continue
            got = torch.autograd.grad([o, S], (q, k, v, g, s0), [s["do"][b, hs, lo:hi].double(), s["ds"][i, hs].double()])
            for name, t in zip(("dq", "dk", "dv"), got):
                out[name][b, hs, lo:hi] = t
            if case["g"] == "head":
                out["dg"][hs] += got[3]
            else:
                out["dg"][b, hs, lo:hi] = got[3]
            if case["state"]:
                out["dstate"][i, hs] = got[4]
    return out
