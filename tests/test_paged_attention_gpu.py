"""causal_attention_step_paged: the same bits as causal_attention_step over a cache of the same places, which is held to its definition in float64
with the bounds of test_attention_gpu.py."""
import pytest
import torch

import linearnexus_amd as la
from test_attention_gpu import DEV, DT, _check_step, _inputs, _step_inputs

pytestmark = pytest.mark.gpu


def _paged(kc, vc, page, lens, *, token_first=False, spare=2, fill=None, seed=0):
    """Pools of pages that hold the places of dense caches ``[B, Hkv, S, d]`` in no order, S a multiple of the page; entries that are not in
    use name no page, pages that are not in use hold NaN."""
    B, Hkv, S, d = kc.shape
    used = [n // page + 1 for n in lens]
    P = sum(used) + spare
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(seed))
    table = torch.full((B, S // page), -1 if fill is None else fill, dtype=torch.int32)
    pools = [torch.full((P, Hkv, page, d), float("nan"), dtype=kc.dtype, device=DEV) for _ in range(2)]
    at = 0
    for b, u in enumerate(used):
        for i in range(u):
            table[b, i] = ids[at]
            for pool, c in zip(pools, (kc, vc)):
                pool[ids[at]] = c[b, :, i * page : (i + 1) * page]
            at += 1
    if token_first:
        pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pools]
    return *pools, table.to(DEV)


def _dense(pool, table, like, lens, page):
    out = like.clone()
    for b, n in enumerate(lens):
        for i in range(n // page + 1):
            out[b, :, i * page : (i + 1) * page] = pool[table[b, i]]
    return out


def _check(q, k, v, kc, vc, lens, page, scale=None, **kw):
    kp, vp, table = _paged(kc, vc, page, lens, **kw)
    keep = [t.clone() for t in (kp, vp, table)]
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = la.causal_attention_step_paged(q, k, v, kp, vp, table, lengths, scale)
    for b, n in enumerate(lens):  # the pools hold the new token and are otherwise as they were
        for pool, new in zip(keep[:2], (k, v)):
            pool[table[b, n // page], :, n % page] = new[b]
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip((kp, vp), keep)) and torch.equal(table, keep[2]) and lengths.tolist() == lens
    want = la.causal_attention_step(q, k, v, kc, vc, lengths, scale)
    assert torch.equal(o, want)
    return kp, vp, table


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("token_first", [False, True])
@pytest.mark.parametrize("page", [1, 3, 16, 24, 31, 32, 33, 48, 64, 100, 128, 200])
def test_pages(page, token_first, dtype):
    n = -(-300 // page)
    lens = [0, n * page - 1, page - 1, min(page, n * page - 1), 170]
    q, k, v, kc, vc = _step_inputs(5, 6, 2, n * page, 64, dtype)
    for b, m in enumerate(lens):  # what lies behind the token is nobody's business
        kc[b, :, m:] = float("nan")
        vc[b, :, m:] = float("nan")
    _check(q, k, v, kc, vc, lens, page, token_first=token_first, fill=1 << 30)
    _check_step(q, k, v, kc, vc, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,Hkv,pages,page,d,lens", [(1, 1, 1, 1, 1, 8, [0]), (3, 6, 2, 3, 11, 128, [31, 32, 5]), (2, 8, 8, 5, 60, 80, [64, 299]), (1, 40, 1, 20, 10, 64, [130]),
                                                       (2, 16, 4, 63, 16, 128, [999, 511]), (1, 8, 2, 47, 64, 128, [2700]), (2, 3, 3, 28, 25, 40, [3, 640])])
def test_shapes(B, H, Hkv, pages, page, d, lens, dtype):
    q, k, v, kc, vc = _step_inputs(B, H, Hkv, pages * page, d, dtype)
    _check(q, k, v, kc, vc, lens, page)
    _check_step(q, k, v, kc, vc, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,pages,page,d,n", [(8, 1094, 64, 128, 69_999), (3, 4375, 16, 64, 2), (40, 800, 25, 40, 17_003), (2, 9000, 1, 128, 8_999)])
def test_many_shares(H, pages, page, d, n, dtype):
    """One key head and a long cache: hundreds of workgroups share the sequence, or find nothing of it."""
    _check(*_step_inputs(1, H, 1, pages * page, d, dtype), [n], page)


@pytest.mark.parametrize("scale", [-0.4, 0.0, 3.0])
def test_scales(scale):
    _check(*_step_inputs(2, 4, 2, 160, 64, "bf16"), [149, 60], 16, scale)


def test_strided_pools_and_tables():
    q, k, v, kc, vc = _step_inputs(2, 4, 2, 96, 64, "bf16")
    lens = [88, 10]
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = la.causal_attention_step(q, k, v, kc.clone(), vc.clone(), lengths)
    kp, vp, table = _paged(kc, vc, 16, lens)
    both = torch.stack([kp, vp], 1)  # [pages, key or value, Hkv, page, d]
    wide = torch.full((2, 40), -7, dtype=torch.int32, device=DEV)
    wide[:, 3:9] = table
    assert torch.equal(la.causal_attention_step_paged(q, k, v, both[:, 0], both[:, 1], wide[:, 3:9], lengths), want)
    assert torch.equal(_dense(both[:, 0], table, kc, lens, 16)[0, :, 88], k[0])


def test_sequences_share_pages():
    """Two sequences with one beginning: its pages are in both rows of the table."""
    q, k, v, kc, vc = _step_inputs(2, 4, 2, 64, 64, "f32")
    kc[1, :, :32], vc[1, :, :32] = kc[0, :, :32], vc[0, :, :32]
    lens = [40, 50]
    kp, vp, table = _paged(kc, vc, 16, lens)
    table[1, :2] = table[0, :2]
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = la.causal_attention_step_paged(q, k, v, kp, vp, table, lengths)
    assert torch.equal(o, la.causal_attention_step(q, k, v, kc, vc, lengths))


def test_no_place_or_no_page_gives_nan_and_writes_nothing_elsewhere():
    q, k, v, kc, vc = _step_inputs(6, 4, 2, 1600, 64, "bf16")
    lens = [900, 900, 900, 900, 900, 900]
    kp, vp, table = _paged(kc, vc, 16, lens)
    table[1, 20] = -1              # a page that is read is none
    table[2, 3] = kp.shape[0]      # one behind the pool
    table[3, 900 // 16] = 1 << 30  # the new token's
    lengths = torch.tensor([900, 900, 900, 900, 1600, -1], dtype=torch.int32, device=DEV)
    k0, v0 = kp.clone(), vp.clone()
    o = la.causal_attention_step_paged(q, k, v, kp, vp, table, lengths)
    assert bool(torch.isfinite(o[0]).all()) and bool(torch.isnan(o[1:]).all())
    for b in (0, 1, 2):
        k0[table[b, 900 // 16], :, 900 % 16], v0[table[b, 900 // 16], :, 900 % 16] = k[b], v[b]
    assert torch.equal(kp.nan_to_num(7.0), k0.nan_to_num(7.0)) and torch.equal(vp.nan_to_num(7.0), v0.nan_to_num(7.0))


def test_pools_beyond_two_to_the_31_elements():
    P, page, d = 2 ** 18 + 3, 64, 128
    kp, vp = (torch.zeros(P, 1, page, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q, k, v, kc, vc = _step_inputs(1, 4, 1, 128, d, "bf16")
    table = torch.tensor([[P - 1, P - 2]], dtype=torch.int32, device=DEV)
    for i in range(2):
        kp[P - 1 - i], vp[P - 1 - i] = kc[0, :, 64 * i : 64 * i + 64], vc[0, :, 64 * i : 64 * i + 64]
    lengths = torch.tensor([100], dtype=torch.int32, device=DEV)
    assert torch.equal(la.causal_attention_step_paged(q, k, v, kp, vp, table, lengths), la.causal_attention_step(q, k, v, kc, vc, lengths))
    assert torch.equal(kp[P - 2, :, 36], k[0]) and not bool(kp[: P - 2].any())


def test_prompt_then_tokens_in_a_replayed_graph():
    """Pages filled from a prompt; the graph's tokens advance the lengths, pages are handed out between replays."""
    q, k, v, _ = _inputs(2, 4, 2, 70, 64, "f32")
    whole = la.causal_attention(q, k, v)
    page, n = 8, 10
    kp, vp = torch.full((25, 2, page, 64), float("nan"), device=DEV), torch.full((25, 2, page, 64), float("nan"), device=DEV)
    order = torch.randperm(25, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(DEV)[:20].view(2, n)
    table = torch.full((2, n), -1, dtype=torch.int32, device=DEV)
    table[:, :8] = order[:, :8]
    for b in range(2):
        for t in range(60):
            kp[order[b, t // page], :, t % page], vp[order[b, t // page], :, t % page] = k[b, :, t], v[b, :, t]
    lengths = torch.full((2,), 60, dtype=torch.int32, device=DEV)
    tok = [t[:, :, 60].clone() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        la.causal_attention_step_paged(*tok, kp, vp, table, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = la.causal_attention_step_paged(*tok, kp, vp, table, lengths)
        lengths.add_(1)
    for t in range(60, 70):
        for buf, x in zip(tok, (q, k, v)):
            buf.copy_(x[:, :, t])
        table[:, t // page] = order[:, t // page]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(o, whole[:, :, t], rtol=1e-5, atol=1e-5)
    assert lengths.tolist() == [70, 70]


def test_counts_as_a_write():
    q, k, v, kc, vc = _step_inputs(1, 4, 2, 32, 64, "f32")
    kp, vp, table = _paged(kc, vc, 16, [5])
    w = torch.ones(1, device=DEV, requires_grad=True)
    out = (w * kp.nan_to_num_(0.0)).sum()
    la.causal_attention_step_paged(q, k, v, kp, vp, table, torch.tensor([5], dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_refusals():
    q, k, v, kc, vc = _step_inputs(2, 4, 2, 32, 64, "f32")
    kp, vp, table = _paged(kc, vc, 8, [9, 9])
    n = torch.tensor([9, 9], dtype=torch.int32, device=DEV)
    call = la.causal_attention_step_paged
    e = torch.zeros(0, 4, 64, device=DEV)
    assert call(e, e[:, :2], e[:, :2], kp, vp, table[:0], n[:0]).shape == (0, 4, 64)
    shared = kp.as_strided(kp.shape, (0, *kp.stride()[1:]))
    for bad in (lambda: call(q, k, v, kp, vp[:, :, :5], table, n), lambda: call(q, k, v, kp, vp, table, n.long()), lambda: call(q, k, v, kp, vp, table.long(), n),
                lambda: call(q, k, v, kp, vp, table[:1], n), lambda: call(q, k, v, kp, vp, table[:, :0], n), lambda: call(q, k, v, kp, vp, table.t(), n),
                lambda: call(q, k, v, kp, vp, table[:, ::2], n), lambda: call(q, k, v, kp, kp, table, n), lambda: call(q, k, v, shared, vp, table, n),
                lambda: call(q, k, v, kp.bfloat16(), vp, table, n), lambda: call(q, k, v, kp, vp, table.cpu(), n), lambda: call(q, k, v, kp[:0], vp[:0], table, n),
                lambda: call(q.requires_grad_(), k, v, kp, vp, table, n)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        call(q.detach(), k, v, kp, vp, table, n, float("inf"))
