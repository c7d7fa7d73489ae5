"""Boundary of decay linear attention, layer norm and the paged attention step without a GPU: argument blocks as the header lays them out,
refusals that happen before anything is dereferenced, workspace sizes, and the Python ops' own checks."""
import ctypes as C
import inspect

import pytest
import torch

import linearnexus_amd as la
from linearnexus_amd import _lib

_keep = []


def _ptr(shift=0):
    buf = (C.c_char * 128)()
    _keep.append(buf)
    return C.c_void_p(((C.addressof(buf) + 63) & ~63) + shift)


def _refused(status, want, text):
    assert status == want and text in _lib.load().lnx_last_error(), (status, _lib.load().lnx_last_error())


def test_argument_blocks():
    # rows, four of four bytes, ten pointers and sizes
    assert _lib.LayerNormArgs.x.offset == 24 and C.sizeof(_lib.LayerNormArgs) == 24 + 10 * 8
    # ten of four bytes, five tensors, six pointers and sizes
    assert _lib.AttnStepPagedArgs.q.offset == 40 and C.sizeof(_lib.AttnStepPagedArgs) == 40 + 5 * 32 + 6 * 8
    # ten of four bytes, eight tensors, thirteen pointers and sizes
    assert _lib.DecayArgs.q.offset == 40 and _lib.DecayArgs.g.offset == 40 + 8 * 32 and C.sizeof(_lib.DecayArgs) == 40 + 8 * 32 + 13 * 8
    assert _lib.DecayStepArgs.q.offset == 24 and C.sizeof(_lib.DecayStepArgs) == 24 + 9 * 8


def test_signatures():
    def names(f):
        return [p.name for p in inspect.signature(f).parameters.values()]

    assert names(la.decay_linear_attention) == ["q", "k", "v", "g", "scale", "initial_state", "cu_seqlens"]
    assert names(la.decay_linear_attention_step) == ["q", "k", "v", "g", "state", "scale", "inplace"]
    assert names(la.layer_norm) == ["x", "weight", "bias", "eps"]
    assert names(la.causal_attention_step_paged) == ["q", "k", "v", "k_pages", "v_pages", "page_table", "lengths", "scale"]
    for n in ("decay_linear_attention", "decay_linear_attention_step", "layer_norm", "causal_attention_step_paged"):
        assert n in la.__all__


def _decay(**kw):
    a = _lib.DecayArgs(**{**dict(B=1, H=4, T=8, dk=64, dv=64, dtype=_lib.LNX_BF16, scale=1.0, g_stride_b=32, g_stride_h=8, g_stride_t=1), **kw})
    for n in ("q", "k", "v", "o", "d_o", "d_q", "d_k", "d_v"):
        setattr(a, n, _lib.Tensor4(_ptr(), 8 * 4 * 64, 8 * 64, 64))
    a.g = a.final_state = a.d_g = _ptr()
    return a


def test_decay_refusals():
    lib = _lib.load()
    for fn, bwd in ((lib.lnx_decay_fwd, False), (lib.lnx_decay_bwd, True)):
        _refused(fn(None, None), -1, b"NULL")
        for kw in (dict(B=-1), dict(H=0), dict(T=-1), dict(T=0x7fffff01), dict(dk=0), dict(dk=257), dict(dv=0), dict(dv=257), dict(nseq=-1), dict(B=2, nseq=1)):
            _refused(fn(_decay(**kw), None), -2, b"dimensions")
        _refused(fn(_decay(dtype=2), None), -3, b"dtype")
        _refused(fn(_decay(nseq=1), None), -1, b"cu_seqlens")
        for bad in (float("nan"), float("inf"), -float("inf")):
            _refused(fn(_decay(scale=bad), None), -2, b"finite")
        for n in ("q", "k", "v", *(("d_o", "d_q", "d_k", "d_v") if bwd else ("o",))):
            a = _decay()
            getattr(a, n).p = None
            _refused(fn(a, None), -1, b"missing")
            a = _decay()
            getattr(a, n).p = _ptr(8)
            _refused(fn(a, None), -2, b"aligned")
            a = _decay()
            getattr(a, n).stride_t = 68
            _refused(fn(a, None), -2, b"aligned")
            a = _decay()
            getattr(a, n).stride_t = -64
            _refused(fn(a, None), -2, b"16 MiB")
            a = _decay()
            getattr(a, n).stride_t = 1 << 24
            _refused(fn(a, None), -2, b"16 MiB")
        a = _decay()
        a.g = None
        _refused(fn(a, None), -1, b"g is required")
        # more workgroups than a launch takes: 512 threads a walk
        _refused(fn(_decay(B=1 << 23, H=1, T=1), None), -2, b"too many rows")
        a = _decay(nseq=1 << 23, H=1, T=1)
        a.cu_seqlens = _ptr()
        _refused(fn(a, None), -2, b"too many rows")
        assert fn(_decay(B=0), None) == 0
    # 1024 threads a row sum up the gates' gradients: what the forward pass takes, the backward pass may not
    a = _decay(B=1 << 22, H=1, T=1)
    _refused(lib.lnx_decay_bwd(a, None), -2, b"too many rows")
    a = _decay()
    a.final_state = None
    _refused(lib.lnx_decay_fwd(a, None), -1, b"final_state")
    a.d_final_state = _ptr()
    _refused(lib.lnx_decay_bwd(a, None), -1, b"final_state")
    a = _decay()
    a.d_g = None
    _refused(lib.lnx_decay_bwd(a, None), -1, b"d_g")
    _refused(lib.lnx_decay_bwd(_decay(), None), -4, b"workspace")
    a = _decay()
    a.workspace, a.workspace_bytes = _ptr(4), 1 << 30
    _refused(lib.lnx_decay_bwd(a, None), -4, b"aligned")
    long = _decay(H=1, T=4096)  # few walks: segments
    _refused(lib.lnx_decay_fwd(long, None), -4, b"workspace")
    _refused(lib.lnx_decay_bwd(long, None), -1, b"kept")


def test_decay_sizes():
    lib = _lib.load()
    kept, fwd, bwd = lib.lnx_decay_kept_bytes, lib.lnx_decay_fwd_workspace_bytes, lib.lnx_decay_bwd_workspace_bytes
    a = _decay(B=1, H=129, T=4096)  # a walk for every CU and more: nothing is kept
    assert kept(a) == 0 and fwd(a) == 0
    assert bwd(a) >= 4 * 129 * 4096 * 4
    # 4096 tokens of one head: 16 segments of 256; fp32: 32 of 128
    for dtype, n in ((_lib.LNX_BF16, 16), (_lib.LNX_F32, 32)):
        a = _decay(H=1, T=4096, dtype=dtype)
        assert kept(a) == n * 64 * 64 * 4 and fwd(a) == kept(a) + n * 4
        a.kept = _ptr()
        assert fwd(a) == n * 4
        assert bwd(a) >= 4 * 4096 * 4 + kept(a) + n * 4
    a = _decay()  # the gradient of an initial state is formed, whether the caller wants it or not
    small = bwd(a)
    a.initial_state = _ptr()
    assert bwd(a) == small + 4 * 64 * 64 * 4
    a.d_initial_state = _ptr()
    assert bwd(a) == small
    assert kept(_decay(H=1, T=512)) == 0 and kept(_decay(H=1, T=513)) == 3 * 64 * 64 * 4
    assert kept(_decay(H=2, T=4096, nseq=5)) == (4096 // 256 + 5) * 2 * 64 * 64 * 4  # a slot more for every sequence
    for bad in (dict(B=0), dict(H=0), dict(dk=0), dict(dv=300), dict(T=-1), dict(nseq=-1)):
        assert kept(_decay(**bad)) == fwd(_decay(**bad)) == bwd(_decay(**bad)) == 0
    assert kept(None) == fwd(None) == bwd(None) == 0


def test_decay_step_refusals():
    lib = _lib.load()

    def step(**kw):
        a = _lib.DecayStepArgs(**{**dict(B=2, H=4, dk=64, dv=64, dtype=_lib.LNX_BF16, scale=1.0), **kw})
        a.q = a.k = a.v = a.g = a.state = a.o = a.new_state = _ptr()
        return a

    _refused(lib.lnx_decay_step(None, None), -1, b"NULL")
    for kw in (dict(B=-1), dict(H=0), dict(dk=0), dict(dk=257), dict(dv=0)):
        _refused(lib.lnx_decay_step(step(**kw), None), -2, b"dimensions")
    _refused(lib.lnx_decay_step(step(dtype=9), None), -3, b"dtype")
    _refused(lib.lnx_decay_step(step(scale=float("nan")), None), -2, b"finite")
    for n in ("q", "k", "v", "g", "state", "o", "new_state"):
        a = step()
        setattr(a, n, None)
        _refused(lib.lnx_decay_step(a, None), -1, b"missing")
    _refused(lib.lnx_decay_step(step(B=1 << 24, H=1), None), -2, b"too many rows")
    assert lib.lnx_decay_step(step(B=0), None) == 0


def test_layer_norm_refusals():
    lib = _lib.load()
    for fn, bwd in ((lib.lnx_layer_norm_fwd, False), (lib.lnx_layer_norm_bwd, True)):
        _refused(fn(None, None), -1, b"NULL")

        def args(**kw):
            a = _lib.LayerNormArgs(**{**dict(rows=4, heads=1, d=8, eps=1e-5, dtype=_lib.LNX_F32), **kw})
            a.x = a.y = a.d_y = a.d_x = _ptr()
            return a

        for kw in (dict(rows=-1), dict(rows=1 << 31), dict(d=0), dict(d=8193), dict(heads=0), dict(heads=3), dict(rows=1 << 17, heads=1 << 17), dict(rows=1 << 14, heads=1 << 14, d=8192)):
            _refused(fn(args(**kw), None), -2, b"rows=")
        _refused(fn(args(dtype=2), None), -3, b"dtype")
        for n in ("x", *(("d_y", "d_x") if bwd else ("y",))):
            a = args()
            setattr(a, n, None)
            _refused(fn(a, None), -1, b"required")
        assert fn(args(rows=0), None) == 0
        if bwd:
            a = args()
            a.d_weight = _ptr()
            _refused(fn(a, None), -4, b"workspace")
            a.workspace, a.workspace_bytes = _ptr(4), 1 << 20
            _refused(fn(a, None), -4, b"aligned")
            a.workspace, a.workspace_bytes = _ptr(), 16
            _refused(fn(a, None), -4, b"workspace")
    size = lib.lnx_layer_norm_bwd_workspace_bytes
    assert size(10, 1, 33, 0) == 1 * 2 * 36 * 4  # 16 rows a workgroup, columns padded to four
    assert size(1 << 20, 1, 2048, 1) == 768 * 2 * 2048 * 4
    assert size(1 << 20, 16, 128, 1) == 768 * 2 * 128 * 4  # of all heads together
    assert size(0, 1, 8, 0) == 2 * 8 * 4
    assert size(-1, 1, 8, 0) == size(8, 0, 8, 0) == size(8, 1, 0, 0) == size(8, 1, 8193, 0) == 0


def test_paged_step_refusals():
    lib = _lib.load()

    def step(**kw):
        a = _lib.AttnStepPagedArgs(**{**dict(B=1, H=4, Hkv=2, d=64, dtype=_lib.LNX_BF16, page=16, pages=3, table_width=2, scale=1.0, table_stride=2), **kw})
        for n in ("q", "k", "v", "k_cache", "v_cache"):
            setattr(a, n, _lib.Tensor4(_ptr(), 4 * 64, 64, 64))
        a.o = a.lengths = a.page_table = _ptr()
        return a

    fn, size = lib.lnx_attn_step_paged, lib.lnx_attn_step_paged_workspace_bytes
    _refused(fn(None, None), -1, b"NULL")
    for kw in (dict(B=-1), dict(H=3), dict(Hkv=0), dict(d=12), dict(d=136), dict(page=0), dict(pages=0), dict(table_width=0), dict(page=1 << 16, table_width=1 << 15)):
        _refused(fn(step(**kw), None), -2, b"dimensions")
    _refused(fn(step(dtype=2), None), -3, b"dtype")
    _refused(fn(step(scale=float("inf")), None), -2, b"finite")
    for n in ("o", "lengths", "page_table"):
        a = step()
        setattr(a, n, None)
        _refused(fn(a, None), -1, b"required")
    for n in ("q", "k", "v", "k_cache", "v_cache"):
        a = step()
        getattr(a, n).p = None
        _refused(fn(a, None), -1, b"missing")
        a = step()
        getattr(a, n).p = _ptr(4)
        _refused(fn(a, None), -2, b"aligned")
    a = step()
    a.k_cache.stride_t = 1 << 24
    _refused(fn(a, None), -2, b"16 MiB")
    _refused(fn(step(table_width=256), None), -4, b"workspace")
    _refused(fn(step(B=1 << 26), None), -2, b"too many rows")
    assert fn(step(B=0), None) == 0 and size(step(B=0)) == 0 and size(None) == 0
    assert size(step(table_width=256)) > 0 == size(step(page=1 << 16, table_width=1 << 15))


def test_tensors_off_the_gpu_are_refused():
    h, g, s = torch.zeros(1, 2, 4, 8), torch.zeros(1, 2, 4), torch.zeros(1, 2, 8, 8)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: la.decay_linear_attention(h, h, h, g), lambda: la.decay_linear_attention_step(h[:, :, 0], h[:, :, 0], h[:, :, 0], g[:, :, 0], s),
                 lambda: la.layer_norm(h), lambda: la.causal_attention_step_paged(h[:, :, 0], h[:, :, 0], h[:, :, 0], h, h, i[None], i)):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: la.decay_linear_attention(h, h, [1.0], g), lambda: la.decay_linear_attention_step(h[:, :, 0], None, h[:, :, 0], g[:, :, 0], s),
                 lambda: la.layer_norm(1.0), lambda: la.causal_attention_step_paged(h[:, :, 0], h[:, :, 0], h[:, :, 0], h, h, None, i)):
        with pytest.raises(TypeError):
            call()
    for bad in ([0, 3], [1, 4], [0, 5, 4]):
        with pytest.raises(ValueError):
            la.decay_linear_attention(h, h, h, g, cu_seqlens=bad)
