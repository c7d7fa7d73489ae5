"""The operators of a hybrid layer stack next to the delta-rule scans -- the element-wise gated recurrence, the norms around
a block on its residual stream, and causal attention with grouped heads -- as cases that can be timed and compared.

``listed()`` gives the fixed cases and ``draw(rng)`` one more of the same ranges; ``prepare`` makes what a program holds
before the call, ``run`` is one pass, ``work`` what that pass cannot do without, and ``exact`` the pass's outputs from the
operators' definitions in 64 bits.  With ``own`` false a pass is the plain form in elementary torch operations in float32,
rounded once at the end; with ``own`` true it is the library's operator as a user calls it.

Kinds of case:

``rec``      gated linear recurrence over ``[B, T, D]``, ``h_t = exp(g_t) h_{t-1} + x_t``, dense or packed; with ``grad`` the
             backward pass too.
``rec_step`` one decode token of it, state in place.
``norm``     ``r' = r + scale sigmoid(gate) RMSNorm(x; post)``, ``z = RMSNorm(r'; weight)``; with ``grad`` the backward pass.
``attn``     causal attention over whole prompts, grouped heads, dense or packed; with ``grad`` the backward pass.
``attn_step`` one decode token against key and value caches of ragged fill: the token is appended, then attends.
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


def _rec(B, T, D, dtype, g_dtype, *, nseq=0, grad, state, name=None):
    c = {"kind": "rec", "B": B, "T": T, "D": D, "dtype": dtype, "g_dtype": g_dtype, "nseq": nseq, "grad": grad, "state": state}
    return c if name is None else {"name": name, **c}


def _norm(rows, d, dtype, r_dtype, *, post, gate, scale, grad, name=None):
    c = {"kind": "norm", "rows": rows, "d": d, "dtype": dtype, "r_dtype": r_dtype, "post": post, "gate": gate, "scale": scale, "grad": grad}
    return c if name is None else {"name": name, **c}


def _attn(B, H, Hkv, T, d, dtype, *, nseq=0, grad, token_first, name=None):
    c = {"kind": "attn", "B": B, "H": H, "Hkv": Hkv, "T": T, "d": d, "dtype": dtype, "nseq": nseq, "grad": grad, "token_first": token_first}
    return c if name is None else {"name": name, **c}


def _step_case(B, H, Hkv, S, d, dtype, name=None):
    c = {"kind": "attn_step", "B": B, "H": H, "Hkv": Hkv, "S": S, "d": d, "dtype": dtype}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # the recurrent mixer of a training step at the repository's headline batch (8 x 4096 tokens, 16 heads of 128)
        _rec(8, 4096, 2048, "bf16", "bf16", grad=True, state=False, name="rec_train"),
        # one very long prompt being prefilled: few channels' worth of parallelism, log-decays in float32, the state kept
        _rec(1, 65536, 2048, "bf16", "f32", grad=False, state=True, name="rec_prompt_t65536"),
        # a small model in float32 on packed documents of ragged length, an odd width
        _rec(1, 5003, 1000, "f32", "f32", nseq=7, grad=True, state=True, name="rec_packed_f32"),
        # one decode token of a server's batch (the repository's decode configuration, 32 heads of 128)
        {"name": "rec_step_b256", "kind": "rec_step", "B": 256, "D": 4096, "dtype": "bf16", "g_dtype": "f32"},
        # the norms around a block in the same training step: norm after the block, its gate, float32 residual stream, norm before the next
        _norm(32768, 2048, "bf16", "f32", post=True, gate=True, scale="number", grad=True, name="norm_train"),
        # an odd number of rows of an odd width on a bf16 stream, a trained scale per channel and no norm behind the block
        _norm(2007, 1000, "bf16", "bf16", post=False, gate=False, scale="channels", grad=True, name="norm_ragged"),
        # one decode token of a small batch: latency
        _norm(27, 4096, "bf16", "f32", post=True, gate=True, scale="number", grad=False, name="norm_token_b27"),
        # the attention layer of a training step, grouped heads, tensors as the projections leave them
        _attn(2, 16, 4, 4096, 128, "bf16", grad=True, token_first=True, name="attn_train"),
        # prompts of different lengths in one packed prefill
        _attn(1, 32, 8, 8192, 128, "bf16", nseq=8, grad=False, token_first=True, name="attn_packed"),
        # a small float32 model's training step at an odd length
        _attn(3, 6, 2, 517, 64, "f32", grad=True, token_first=False, name="attn_f32_t517"),
        # one decode token of a server's batch against long caches
        _step_case(32, 32, 8, 8192, 128, "bf16", name="attn_step_b32"),
        # one user's decode token, a short odd cache: latency
        _step_case(1, 16, 4, 1000, 128, "bf16", name="attn_step_b1"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["rec", "rec", "rec_step", "norm", "norm", "attn", "attn", "attn_step"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    grad = rng.random() < 0.5
    if kind == "rec":
        D, T = _log(rng, 64, 8192), _log(rng, 1, 65536)
        T = max(1, min(T, (1 << 25) // D))
        B = max(1, min(_log(rng, 1, 16), (1 << 25) // (D * T)))
        nseq = rng.randint(1, min(T, 24)) if rng.random() < 0.4 else 0
        return _rec(1 if nseq else B, T, D, dtype, rng.choice([dtype, "f32"]), nseq=nseq, grad=grad, state=rng.random() < 0.5)
    if kind == "rec_step":
        return {"kind": kind, "B": _log(rng, 1, 256), "D": _log(rng, 64, 4096), "dtype": dtype, "g_dtype": rng.choice([dtype, "f32"])}
    if kind == "norm":
        d = _log(rng, 64, 8192)
        rows = max(1, min(_log(rng, 1, 32768), (1 << 25) // d))
        return _norm(rows, d, dtype, rng.choice([dtype, "f32"]), post=rng.random() < 0.6, gate=rng.random() < 0.6, scale=rng.choice(["number", "channels"]), grad=grad)
    Hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 128, 128, 80, 40])
    if kind == "attn":
        T = _log(rng, 1, 4096)
        most = (1 << 29) if dtype == "bf16" else (1 << 26)  # pairs of query and key: a float32 product costs ten times as much
        H = Hkv * group
        if H * T * T > most:
            T = max(1, int(math.sqrt(most / H)))
        B = max(1, min(_log(rng, 1, 8), most // (H * T * T)))
        nseq = rng.randint(1, min(T, 12)) if rng.random() < 0.4 else 0
        return _attn(1 if nseq else B, H, Hkv, T, d, dtype, nseq=nseq, grad=grad, token_first=rng.random() < 0.5)
    S = _log(rng, 1, 8192)
    B = max(1, min(_log(rng, 1, 64), (1 << 24) // (Hkv * S * max(1, d // 16))))
    return _step_case(B, Hkv * group, Hkv, S, d, dtype)


def _lengths(case, seed):
    """Lengths of the packed sequences, at least one token each, summing to T: the same for every seed of a case, as `work` needs them."""
    r = random.Random(case["nseq"] * 1000003 + case["T"])
    cuts = sorted(r.sample(range(1, case["T"]), case["nseq"] - 1))
    return [b - a for a, b in zip([0, *cuts], [*cuts, case["T"]])]


def _fills(case):
    """Tokens that each cache of a decode batch already holds: ragged, between half of the places and all but the last."""
    r = random.Random(case["B"] * 1000003 + case["S"])
    return [r.randint((case["S"] - 1) // 2, case["S"] - 1) for _ in range(case["B"])]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def n(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std).to(dtype)

    def decay(*shape):
        # log-decays as a trained gate gives them: time constants from one token to a thousand, spread over the channels
        rate = torch.exp(torch.rand(shape[-1], generator=gen, device=DEVICE) * math.log(1000.0)).reciprocal()
        z = torch.randn(*shape, generator=gen, device=DEVICE)
        return (-rate * torch.nn.functional.softplus(z + 0.5)).to(DTYPES[case["g_dtype"]])

    s = {"case": case}
    if case["kind"] in ("rec", "rec_step"):
        if case["kind"] == "rec_step":
            s.update(x=n(case["B"], case["D"]), g=decay(case["B"], case["D"]), state=n(case["B"], case["D"], dtype=torch.float32))
            return s
        B, T, D = case["B"], case["T"], case["D"]
        s.update(x=n(B, T, D), g=decay(B, T, D), state=None, cu=None, lens=None)
        rows = B
        if case["nseq"]:
            s["lens"], rows = _lengths(case, seed), case["nseq"]
            s["cu"] = torch.tensor([0, *torch.tensor(s["lens"]).cumsum(0).tolist()], dtype=torch.int32, device=DEVICE)
        if case["state"]:
            s["state"] = n(rows, D, dtype=torch.float32)
        if case["grad"]:
            s.update(dy=n(B, T, D), ds=n(rows, D, std=0.1, dtype=torch.float32))
    elif case["kind"] == "norm":
        rows, d = case["rows"], case["d"]
        s.update(x=n(rows, d), r=n(rows, d, std=3.0, dtype=DTYPES[case["r_dtype"]]), w=1 + n(d, std=0.2, dtype=torch.float32), post=None, gate=None, scale=0.5)
        if case["post"]:
            s["post"] = 1 + n(d, std=0.2, dtype=torch.float32)
        if case["gate"]:
            s["gate"] = n(rows, d)
        if case["scale"] == "channels":
            s["scale"] = 0.3 + n(d, std=0.1, dtype=torch.float32)
        if case["grad"]:
            s.update(dz=n(rows, d), dr=n(rows, d, dtype=DTYPES[case["r_dtype"]]))
    elif case["kind"] == "attn":
        B, H, Hkv, T, d = (case[k] for k in ("B", "H", "Hkv", "T", "d"))

        def heads(h, std=1.0):
            return n(B, T, h, d, std=std).transpose(1, 2) if case["token_first"] else n(B, h, T, d, std=std)

        s.update(q=heads(H, 1.5), k=heads(Hkv), v=heads(Hkv), cu=None, lens=None)
        if case["nseq"]:
            s["lens"] = _lengths(case, seed)
            s["cu"] = torch.tensor([0, *torch.tensor(s["lens"]).cumsum(0).tolist()], dtype=torch.int32, device=DEVICE)
        if case["grad"]:
            s["do"] = heads(H)
    else:
        B, H, Hkv, S, d = (case[k] for k in ("B", "H", "Hkv", "S", "d"))
        s.update(q=n(B, H, d, std=1.5), k=n(B, Hkv, d), v=n(B, Hkv, d), kc=n(B, Hkv, S, d), vc=n(B, Hkv, S, d),
                 fill=torch.tensor(_fills(case), dtype=torch.int32, device=DEVICE))
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------

def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 by doubling: every step joins spans of twice the length."""
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _rec_plain(s):
    x, g, cu = s["x"], s["g"], s["cu"]
    B, T, D = x.shape
    a, b = torch.exp(g.float()), x.float()
    first = torch.zeros(T, dtype=torch.bool, device=x.device)
    if cu is None:
        first[0] = True
        where = (slice(None), 0)
        last = (slice(None), T - 1)
    else:
        starts, ends = cu[:-1].long(), cu[1:].long() - 1
        first[starts] = True
        where, last = (0, starts), (0, ends)
    inner = torch.where(first[None, :, None], torch.zeros_like(a), a)
    h0 = torch.zeros_like(b[where]) if s["state"] is None else s["state"].float()
    b = b.clone()
    b[where] = b[where] + a[where] * h0
    h = _scan(inner, b)
    out = {"y": h.to(x.dtype), "state": h[last].clone()}
    if "dy" not in s:
        return out
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    before[where] = h0
    dy = s["dy"].float().clone()
    dy[last] = dy[last] + s["ds"]
    coming = torch.cat([inner[:, 1:], torch.zeros_like(inner[:, :1])], 1)
    dh = _scan(coming.flip(1), dy.flip(1)).flip(1)
    out.update(dx=dh.to(x.dtype), dg=(a * before * dh).to(g.dtype))
    if s["state"] is not None:
        out["dstate"] = a[where] * dh[where]
    return out


def _rec_own(s):
    import linearnexus_amd as la
    if "dy" not in s:
        y, state = la.gated_linear_recurrence(s["x"], s["g"], s["state"], cu_seqlens=s["cu"])
        return {"y": y, "state": state}
    leaves = [t.detach().requires_grad_() for t in (s["x"], s["g"], s["state"]) if t is not None]
    y, state = la.gated_linear_recurrence(*leaves, cu_seqlens=s["cu"])
    grads = torch.autograd.grad([y, state], leaves, [s["dy"], s["ds"]])
    return {"y": y.detach(), "state": state.detach(), **dict(zip(("dx", "dg", "dstate"), grads))}


def _rec_step(s):
    if own:
        import linearnexus_amd as la
        y, state = la.gated_linear_recurrence_step(s["x"], s["g"], s["state"])
        return {"y": y, "state": state}
    h = torch.exp(s["g"].float()) * s["state"] + s["x"].float()
    return {"y": h.to(s["x"].dtype), "state": h}


def _norm_plain(s):
    x, r, w = s["x"].float(), s["r"].float(), s["w"]
    dt, rt = s["x"].dtype, s["r"].dtype
    rho = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) if s["post"] is not None else None
    xn = x if rho is None else x * rho
    post = s["post"] if rho is not None else torch.ones_like(w)
    sg = 1.0 if s["gate"] is None else torch.sigmoid(s["gate"].float())
    out = r + xn * post * sg * s["scale"]
    rho2 = torch.rsqrt((out * out).mean(-1, keepdim=True) + EPS)
    res = {"z": (out * rho2 * w).to(dt), "r": out.to(rt)}
    if "dz" not in s:
        return res
    dz = s["dz"].float()
    u = dz * w
    D = s["dr"].float() + rho2 * (u - out * rho2 * rho2 * (u * out).mean(-1, keepdim=True))
    res["dres"] = D.to(rt)
    res["dw"] = (dz * out * rho2).sum(0)
    both = (D * xn * sg).sum(0)
    u = D * post * sg * s["scale"]
    res["dx"] = (u if rho is None else rho * (u - x * rho * rho * (u * x).mean(-1, keepdim=True))).to(dt)
    if s["post"] is not None:
        res["dpost"] = both * s["scale"]
    if s["gate"] is not None:
        res["dgate"] = (D * xn * post * s["scale"] * sg * (1 - sg)).to(dt)
    if isinstance(s["scale"], torch.Tensor):
        res["dscale"] = both * post
    return res


def _norm_own(s):
    import linearnexus_amd as la
    if "dz" not in s:
        z, r = la.rmsnorm_residual(s["x"], s["r"], s["w"], s["post"], s["gate"], s["scale"], EPS)
        return {"z": z, "r": r}
    leaf = {k: s[k].detach().requires_grad_() for k in ("x", "r", "w", "post", "gate", "scale") if isinstance(s[k], torch.Tensor)}
    z, r = la.rmsnorm_residual(leaf["x"], leaf["r"], leaf["w"], leaf.get("post"), leaf.get("gate"), leaf.get("scale", s["scale"]), EPS)
    grads = dict(zip(leaf, torch.autograd.grad([z, r], list(leaf.values()), [s["dz"], s["dr"]])))
    names = {"x": "dx", "r": "dres", "w": "dw", "post": "dpost", "gate": "dgate", "scale": "dscale"}
    order = ("r", "w", "x", "post", "gate", "scale")
    return {"z": z.detach(), "r": r.detach(), **{names[k]: grads[k] for k in order if k in grads}}


def _attn_plain(s):
    case, cu = s["case"], s["cu"]
    B, H, Hkv, T, d = (case[k] for k in ("B", "H", "Hkv", "T", "d"))
    G, dt, scale = H // Hkv, s["q"].dtype, d ** -0.5
    q = s["q"].float().reshape(B, Hkv, G * T, d)  # the query heads of a key head, one after the other
    k, v = s["k"].float().contiguous(), s["v"].float().contiguous()
    pos = torch.arange(T, device=q.device)
    keep = pos[:, None] >= pos[None, :]
    if cu is not None:
        seq = torch.searchsorted(cu[1:].contiguous(), pos.to(torch.int32), right=True)
        keep = keep & (seq[:, None] == seq[None, :])
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hkv, G, T, T) * scale
    sc = sc.masked_fill_(~keep, float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, Hkv, G * T, T)
    del sc
    o = torch.matmul(p, v)
    out = {"o": o.view(B, H, T, d).to(dt)}
    if "do" not in s:
        return out
    do = s["do"].float().reshape(B, Hkv, G * T, d)
    out["dv"] = torch.matmul(p.transpose(2, 3), do).to(dt)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (o * do).sum(-1, keepdim=True)) * scale
    del dp, p
    out["dq"] = torch.matmul(ds, k).view(B, H, T, d).to(dt)
    out["dk"] = torch.matmul(ds.transpose(2, 3), q).to(dt)
    return out


def _attn_own(s):
    import linearnexus_amd as la
    if "do" not in s:
        return {"o": la.causal_attention(s["q"], s["k"], s["v"], cu_seqlens=s["cu"])}
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o = la.causal_attention(*leaves, cu_seqlens=s["cu"])
    dq, dk, dv = torch.autograd.grad(o, leaves, s["do"])
    return {"o": o.detach(), "dv": dv, "dq": dq, "dk": dk}


def _attn_step(s):
    case = s["case"]
    B, H, Hkv, S, d = (case[k] for k in ("B", "H", "Hkv", "S", "d"))
    if own:
        import linearnexus_amd as la
        o = la.causal_attention_step(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["fill"])
        return {"o": o, "k": s["kc"], "v": s["vc"]}
    row, at = torch.arange(B, device=s["q"].device), s["fill"].long()
    s["kc"][row, :, at] = s["k"]
    s["vc"][row, :, at] = s["v"]
    q = s["q"].float().view(B, Hkv, H // Hkv, d) * d ** -0.5
    sc = torch.matmul(q, s["kc"].float().transpose(2, 3).contiguous())
    sc = sc.masked_fill_((torch.arange(S, device=q.device) > at[:, None])[:, None, None], float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p / p.sum(-1, keepdim=True), s["vc"].float())
    return {"o": o.reshape(B, H, d).to(s["q"].dtype), "k": s["kc"], "v": s["vc"]}


def run(state):
    kind = state["case"]["kind"]
    if kind == "rec_step":
        return _rec_step(state)
    if kind == "attn_step":
        return _attn_step(state)
    if kind == "rec":
        return _rec_own(state) if own else _rec_plain(state)
    if kind == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    return _attn_own(state) if own else _attn_plain(state)


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind in ("rec", "rec_step"):
        n, rows, ge = case["B"] * case.get("T", 1) * case["D"], case["nseq"] or case["B"] if kind == "rec" else case["B"], SIZE[case["g_dtype"]]
        states = rows * case["D"] * 4
        grad = case.get("grad", False)
        has = kind == "rec_step" or case["state"]
        moved = n * (2 * e + ge) + states * (1 + has)  # x, g, y; the states
        if grad:
            moved += n * (2 * e + ge) + states * (1 + has)  # dy, dx, dg; the states' gradients
        return {"bytes": moved, "flops": n * (8 if grad else 3)}
    if kind == "norm":
        rows, d, re = case["rows"], case["d"], SIZE[case["r_dtype"]]
        vectors = 1 + case["post"] + (case["scale"] == "channels")
        moved = rows * d * (2 * e + 2 * re + e * case["gate"]) + 4 * d * vectors  # x, z, r, r', the gate
        if case["grad"]:
            moved += rows * d * (2 * e + 2 * re + e * case["gate"]) + 4 * d * vectors  # dz, dx, dr', dr, the gate's
        return {"bytes": moved, "flops": rows * d * (40 if case["grad"] else 12)}
    B, H, Hkv, d = (case[k] for k in ("B", "H", "Hkv", "d"))
    if kind == "attn":
        T = case["T"]
        pairs = sum(n * (n + 1) // 2 for n in _lengths(case, 0)) if case["nseq"] else B * (T * (T + 1) // 2)
        rows = B * T * d * e
        moved = rows * (2 * H + 2 * Hkv)
        if case["grad"]:
            moved += rows * (2 * H + 2 * Hkv)
        return {"bytes": moved, "flops": pairs * H * d * (14 if case["grad"] else 4)}
    keys = sum(n + 1 for n in _fills(case))
    return {"bytes": keys * Hkv * d * e * 2 + B * (2 * H + 4 * Hkv) * d * e, "flops": keys * H * d * 4}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rec_step":
        h = s["state"].double() * s["g"].double().exp() + s["x"].double()
        return {"y": h, "state": h}
    if kind == "rec":
        return _rec_exact(case, s)
    if kind == "norm":
        return _norm_exact(s)
    if kind == "attn":
        return _attn_exact(case, s)
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["H"] // case["Hkv"]
    for b, fill in enumerate(s["fill"].tolist()):
        for h in range(case["H"]):
            kept = [torch.cat([c[b, h // group, :fill], t[b, h // group][None]]).double() for c, t in ((s["kc"], s["k"]), (s["vc"], s["v"]))]
            o[b, h] = torch.softmax(kept[0] @ s["q"][b, h].double() / math.sqrt(case["d"]), 0) @ kept[1]
    return {"o": o, "k": None, "v": None}


def _rec_exact(case, s):
    """Token by token; all the rows, or all the packed sequences, side by side."""
    lens = s["lens"] or [case["T"]] * case["B"]
    rows, T, D = len(lens), max(lens), case["D"]
    if T * (2 if case["grad"] else 1) * 60e-6 + rows * T * D * 1e-9 > 15:
        return None
    begin = [sum(lens[:i]) for i in range(rows)]

    def unpack(t, fill=0.0):  # [T, rows, D]
        u = torch.full((T, rows, D), fill, dtype=torch.float64, device=t.device)
        for i in range(rows):
            u[: lens[i], i] = t[0, begin[i] : begin[i] + lens[i]] if s["lens"] else t[i]
        return u

    def packed(u):
        return torch.cat([u[: lens[i], i] for i in range(rows)])[None] if s["lens"] else u.transpose(0, 1)

    x, a = unpack(s["x"]), unpack(s["g"]).exp()  # behind a short sequence's end: x = 0, a = 1, the state stands
    h = torch.zeros(rows, D, dtype=torch.float64, device=x.device) if s["state"] is None else s["state"].double()
    h0, ys = h, torch.empty_like(x)
    for t in range(T):
        h = torch.addcmul(x[t], a[t], h, out=ys[t])
    out = {"y": packed(ys), "state": h.clone()}
    if not case["grad"]:
        return out
    dy, dh, dhs = unpack(s["dy"]), s["ds"].double(), torch.empty_like(x)
    for t in range(T - 1, -1, -1):
        torch.add(dy[t], dh, out=dhs[t])
        dh = a[t] * dhs[t]
    before = torch.cat([h0[None], ys[:-1]])
    out.update(dx=packed(dhs), dg=packed(a * before * dhs))
    if s["state"] is not None:
        out["dstate"] = dh
    return out


def _norm_exact(s):
    """The outputs in float64, the gradients by automatic differentiation of them."""
    leaf = {k: s[k].double().requires_grad_() for k in ("r", "w", "x", "post", "gate", "scale") if isinstance(s[k], torch.Tensor)}
    u = leaf["x"]
    if "post" in leaf:
        u = u / torch.sqrt(u.square().mean(1, True) + EPS) * leaf["post"]
    if "gate" in leaf:
        u = u / (1 + torch.exp(-leaf["gate"]))
    r = leaf["r"] + leaf.get("scale", s["scale"]) * u
    z = r / torch.sqrt(r.square().mean(1, True) + EPS) * leaf["w"]
    out = {"z": z.detach(), "r": r.detach()}
    if "dz" in s:
        names = {"x": "dx", "r": "dres", "w": "dw", "post": "dpost", "gate": "dgate", "scale": "dscale"}
        grads = torch.autograd.grad([z, r], list(leaf.values()), [s["dz"].double(), s["dr"].double()])
        out.update({names[k]: g for k, g in zip(leaf, grads)})
    return out


def _attn_exact(case, s):
    """One sequence and one head at a time, the gradients by automatic differentiation."""
    group, out = case["H"] // case["Hkv"], {}
    shape = {"o": s["q"], "dq": s["q"], "dk": s["k"], "dv": s["v"]}
    for name in ("o", "dv", "dq", "dk") if case["grad"] else ("o",):
        out[name] = torch.zeros(shape[name].shape, dtype=torch.float64, device=DEVICE)
    ends = [sum(s["lens"][: i + 1]) for i in range(case["nseq"])] if case["nseq"] else [case["T"]]
    for b in range(case["B"]):
        for lo, hi in zip([0, *ends], ends):
            hide = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=DEVICE).triu(1)
            for h in range(case["H"]):
                q, k, v = (t[b, i, lo:hi].double().requires_grad_(case["grad"]) for t, i in ((s["q"], h), (s["k"], h // group), (s["v"], h // group)))
                o = torch.softmax((q @ k.mT / math.sqrt(case["d"])).masked_fill(hide, -math.inf), 1) @ v
                out["o"][b, h, lo:hi] = o.detach()
                if case["grad"]:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"][b, h, lo:hi].double())
                    out["dq"][b, h, lo:hi] = dq
                    out["dk"][b, h // group, lo:hi] += dk
                    out["dv"][b, h // group, lo:hi] += dv
    return out
