"""Boundary of the recurrence, residual-norm and attention ops without a GPU: argument blocks as the header lays them out, refusals that
happen before anything is dereferenced, workspace sizes, and the Python ops' own checks."""
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
    # six int32, six strides, nine pointers and sizes, five pointers
    assert _lib.LinrecArgs.x_stride_b.offset == 24 and _lib.LinrecArgs.x.offset == 72 and C.sizeof(_lib.LinrecArgs) == 72 + 14 * 8
    assert _lib.RmsnormResidualArgs.x.offset == 32 and C.sizeof(_lib.RmsnormResidualArgs) == 32 + 18 * 8
    assert C.sizeof(_lib.Tensor4) == 32 and _lib.AttnArgs.q.offset == 32 and C.sizeof(_lib.AttnArgs) == 32 + 8 * 32 + 5 * 8
    assert _lib.AttnStepArgs.q.offset == 32 and C.sizeof(_lib.AttnStepArgs) == 32 + 5 * 32 + 4 * 8


def test_signatures():
    def names(f):
        return [p.name for p in inspect.signature(f).parameters.values()]

    assert names(la.gated_linear_recurrence) == ["x", "g", "initial_state", "cu_seqlens"]
    assert names(la.gated_linear_recurrence_step) == ["x", "g", "state", "inplace"]
    assert names(la.rmsnorm_residual) == ["x", "residual", "weight", "post_weight", "gate", "scale", "eps"]
    assert names(la.causal_attention) == ["q", "k", "v", "scale", "cu_seqlens"]
    assert names(la.causal_attention_step) == ["q", "k", "v", "k_cache", "v_cache", "lengths", "scale"]
    for n in ("gated_linear_recurrence", "gated_linear_recurrence_step", "rmsnorm_residual", "causal_attention", "causal_attention_step"):
        assert n in la.__all__


def test_recurrence_refusals():
    lib = _lib.load()
    for fn in (lib.lnx_linrec_fwd, lib.lnx_linrec_bwd):
        _refused(fn(None, None), -1, b"NULL")
        a = _lib.LinrecArgs()
        _refused(fn(a, None), -2, b"dimensions")  # D = 0
        a.B, a.T, a.D, a.dtype = 1, 4, 8, 5
        _refused(fn(a, None), -3, b"dtype")
        a.dtype, a.g_dtype = _lib.LNX_F32, _lib.LNX_BF16
        _refused(fn(a, None), -3, b"dtype")  # a bf16 gate beside fp32
        a.g_dtype = _lib.LNX_F32
        _refused(fn(a, None), -1, b"required")
        a.nseq = 2
        _refused(fn(a, None), -1, b"cu_seqlens")
        a.B = 2
        _refused(fn(a, None), -2, b"dimensions")  # packed batches have one row
    a = _lib.LinrecArgs(B=1, T=4, D=8, x_stride_t=8, g_stride_t=1 << 22)
    a.x = a.g = a.y = a.final_state = _ptr()
    _refused(lib.lnx_linrec_fwd(a, None), -2, b"apart")
    a = _lib.LinrecArgs(B=1, T=8192, D=64, x_stride_t=64, g_stride_t=64)
    a.x = a.g = a.y = a.final_state = _ptr()
    assert lib.lnx_linrec_workspace_bytes(a) > 0
    _refused(lib.lnx_linrec_fwd(a, None), -4, b"workspace")
    a.B = 0
    assert lib.lnx_linrec_fwd(a, None) == 0 and lib.lnx_linrec_workspace_bytes(a) == 0 and lib.lnx_linrec_kept_bytes(a) == 0
    assert lib.lnx_linrec_kept_bytes(_lib.LinrecArgs(B=3, T=257, D=5)) == 3 * 3 * 5 * 4
    assert lib.lnx_linrec_kept_bytes(_lib.LinrecArgs(B=1, T=1000, D=5, nseq=7)) == (1000 // 128 + 7) * 5 * 4
    assert lib.lnx_linrec_step(None, None, None, None, None, 0, 0, 0, None) == 0
    _refused(lib.lnx_linrec_step(None, None, None, None, None, 4, 0, 0, None), -1, b"required")
    _refused(lib.lnx_linrec_step(None, None, None, None, None, -1, 0, 0, None), -2, b"n=-1")
    _refused(lib.lnx_linrec_step(None, None, None, None, None, 4, 0, 1, None), -3, b"dtype")


def test_residual_norm_refusals():
    lib = _lib.load()
    for fn in (lib.lnx_rmsnorm_residual_fwd, lib.lnx_rmsnorm_residual_bwd):
        _refused(fn(None, None), -1, b"NULL")
        a = _lib.RmsnormResidualArgs(rows=2)
        _refused(fn(a, None), -2, b"d=0")
        a.d = 8193
        _refused(fn(a, None), -2, b"8192")
        a.d, a.dtype, a.r_dtype = 8, _lib.LNX_F32, _lib.LNX_BF16
        _refused(fn(a, None), -3, b"dtype")
        a.r_dtype = _lib.LNX_F32
        _refused(fn(a, None), -1, b"x is required")
        a.x = _ptr()
        _refused(fn(a, None), -1, b"required")
    a.d_x = a.d_weight = _ptr()
    _refused(lib.lnx_rmsnorm_residual_bwd(a, None), -4, b"workspace")
    a.d_weight, a.gate = None, _ptr()
    _refused(lib.lnx_rmsnorm_residual_bwd(a, None), -1, b"d_gate")
    a = _lib.RmsnormResidualArgs(rows=0, d=8)
    assert lib.lnx_rmsnorm_residual_fwd(a, None) == 0 and lib.lnx_rmsnorm_residual_bwd(a, None) == 0
    assert lib.lnx_rmsnorm_residual_bwd_workspace_bytes(10, 33, 0) == 3 * 2 * 36 * 4  # four rows a workgroup, columns padded to four
    assert lib.lnx_rmsnorm_residual_bwd_workspace_bytes(1 << 20, 2048, 1) == 768 * 2 * 2048 * 4


def _attn(**kw):
    a = _lib.AttnArgs(**{**dict(B=1, H=4, Hkv=2, T=8, d=64, dtype=_lib.LNX_BF16, scale=1.0), **kw})
    for n in ("q", "k", "v", "o", "d_o", "d_q", "d_k", "d_v"):
        setattr(a, n, _lib.Tensor4(_ptr(), 8 * 4 * 64, 8 * 64, 64))
    return a


def test_attention_refusals():
    lib = _lib.load()
    for fn in (lib.lnx_attn_fwd, lib.lnx_attn_bwd):
        _refused(fn(None, None), -1, b"NULL")
        for kw in (dict(H=3), dict(Hkv=0), dict(d=0), dict(d=136), dict(d=60), dict(B=-1), dict(T=-1), dict(B=2, nseq=1)):
            _refused(fn(_attn(**kw), None), -2, b"dimensions")
        _refused(fn(_attn(dtype=7), None), -3, b"dtype")
        _refused(fn(_attn(nseq=1), None), -1, b"cu_seqlens")
        for bad in (float("nan"), float("inf")):
            _refused(fn(_attn(scale=bad), None), -2, b"finite")
        a = _attn()
        a.k.p = None
        _refused(fn(a, None), -1, b"missing")
        a = _attn()
        a.v.p = _ptr(8)
        _refused(fn(a, None), -2, b"aligned")
        a = _attn()
        a.q.stride_t = 68
        _refused(fn(a, None), -2, b"aligned")
        a = _attn()
        a.q.stride_t = 1 << 24
        _refused(fn(a, None), -2, b"16 MiB")
        assert fn(_attn(B=0), None) == 0 and fn(_attn(T=0), None) == 0
    _refused(lib.lnx_attn_bwd(_attn(), None), -1, b"lse")
    a = _attn()
    a.lse = _ptr()
    _refused(lib.lnx_attn_bwd(a, None), -4, b"workspace")
    assert lib.lnx_attn_bwd_workspace_bytes(_attn()) >= 4 * 8 * 4 and lib.lnx_attn_fwd_workspace_bytes(_attn()) == 0
    long = _attn(B=1, H=1, Hkv=1, T=65536)  # few workgroups: split
    assert lib.lnx_attn_fwd_workspace_bytes(long) > 0
    _refused(lib.lnx_attn_fwd(long, None), -4, b"workspace")
    assert lib.lnx_attn_fwd_workspace_bytes(None) == 0 and lib.lnx_attn_bwd_workspace_bytes(_attn(B=0)) == 0


def test_attention_step_refusals():
    lib = _lib.load()

    def step(**kw):
        a = _lib.AttnStepArgs(**{**dict(B=1, H=4, Hkv=2, S=40, d=64, dtype=_lib.LNX_BF16, scale=1.0), **kw})
        for n in ("q", "k", "v", "k_cache", "v_cache"):
            setattr(a, n, _lib.Tensor4(_ptr(), 4 * 64, 64, 64))
        a.o = a.lengths = _ptr()
        return a

    _refused(lib.lnx_attn_step(None, None), -1, b"NULL")
    for kw in (dict(H=3), dict(S=0), dict(d=12), dict(d=256), dict(B=-1)):
        _refused(lib.lnx_attn_step(step(**kw), None), -2, b"dimensions")
    _refused(lib.lnx_attn_step(step(dtype=2), None), -3, b"dtype")
    _refused(lib.lnx_attn_step(step(scale=float("inf")), None), -2, b"finite")
    a = step()
    a.lengths = None
    _refused(lib.lnx_attn_step(a, None), -1, b"lengths")
    a = step()
    a.k_cache.p = _ptr(4)
    _refused(lib.lnx_attn_step(a, None), -2, b"aligned")
    a = step()
    a.o = _ptr(8)
    _refused(lib.lnx_attn_step(a, None), -2, b"aligned")
    _refused(lib.lnx_attn_step(step(S=4096), None), -4, b"workspace")
    assert lib.lnx_attn_step(step(B=0), None) == 0 and lib.lnx_attn_step_workspace_bytes(step(B=0)) == 0


def test_more_than_a_launch_takes_is_refused():
    lib = _lib.load()
    a = _lib.LinrecArgs(B=1 << 24, T=1, D=64, x_stride_t=64, g_stride_t=64)
    a.x = a.g = a.y = a.final_state = _ptr()
    _refused(lib.lnx_linrec_fwd(a, None), -2, b"too many rows")
    p = _ptr()
    _refused(lib.lnx_linrec_step(p, p, p, p, p, (1 << 32) + 1, 0, 0, None), -2, b"too large")
    _refused(lib.lnx_linrec_step(p, p, p, p, p, 1 << 36, 0, 0, None), -2, b"too large")
    _refused(lib.lnx_attn_fwd(_attn(B=1 << 22, T=1), None), -2, b"too many rows")
    s = _lib.AttnStepArgs(B=1 << 26, H=4, Hkv=4, S=8, d=64, dtype=_lib.LNX_BF16, scale=1.0)
    for n in ("q", "k", "v", "k_cache", "v_cache"):
        setattr(s, n, _lib.Tensor4(_ptr(), 4 * 64, 64, 64))
    s.o = s.lengths = _ptr()
    _refused(lib.lnx_attn_step(s, None), -2, b"too many rows")
    a = _attn()
    a.lse, a.workspace, a.workspace_bytes = _ptr(), _ptr(4), 1 << 20
    _refused(lib.lnx_attn_bwd(a, None), -4, b"aligned")
    n = _lib.RmsnormResidualArgs(rows=2, d=8)
    n.x = n.d_x = n.d_weight = _ptr()
    n.workspace, n.workspace_bytes = _ptr(4), 1 << 20
    _refused(lib.lnx_rmsnorm_residual_bwd(n, None), -4, b"aligned")


def test_tensors_off_the_gpu_are_refused():
    x, v = torch.zeros(1, 4, 8), torch.ones(8)
    h = torch.zeros(1, 2, 4, 8)
    for call in (lambda: la.gated_linear_recurrence(x, x), lambda: la.gated_linear_recurrence_step(x[:, 0], x[:, 0], x[:, 0]), lambda: la.rmsnorm_residual(x, x, v),
                 lambda: la.causal_attention(h, h, h), lambda: la.causal_attention_step(h[:, :, 0], h[:, :, 0], h[:, :, 0], h, h, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: la.gated_linear_recurrence([1.0], x), lambda: la.rmsnorm_residual(x, 1.0, v), lambda: la.causal_attention(h, h, None)):
        with pytest.raises(TypeError):
            call()
    for bad in ([0, 3], [1, 4], [0, 5, 4]):
        with pytest.raises(ValueError):
            la.gated_linear_recurrence(x, x, cu_seqlens=bad)
        with pytest.raises(ValueError):
            la.causal_attention(h, h, h, cu_seqlens=bad)
