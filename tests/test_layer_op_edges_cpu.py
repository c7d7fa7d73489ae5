"""Strides of dimensions of one element at the C boundary, and the records of the kernels' traffic, without a GPU.  Every call below is
refused for another reason behind the strides' check, so that nothing is launched."""
import json
import os

from conftest import ROOT
from linearnexus_amd import _lib
from test_layer_ops_cpu import _attn, _ptr, _refused

ODD = 644  # elements of two bytes: no whole number of 16 bytes


def test_attention_strides_of_single_elements():
    lib = _lib.load()
    long = _attn(H=1, Hkv=1, T=65536)  # needs a workspace, and has none
    for n in ("q", "k", "v", "o"):
        setattr(long, n, _lib.Tensor4(_ptr(), ODD, ODD, 64))
    _refused(lib.lnx_attn_fwd(long, None), -4, b"workspace")
    long.k.stride_t = ODD
    _refused(lib.lnx_attn_fwd(long, None), -2, b"aligned")
    one = _attn(B=2, H=2, Hkv=2, T=1)
    one.lse = _ptr()
    for n in ("q", "k", "v", "o", "d_o", "d_q", "d_k", "d_v"):
        setattr(one, n, _lib.Tensor4(_ptr(), 128, 64, (1 << 40) + 1))
    _refused(lib.lnx_attn_bwd(one, None), -4, b"workspace")
    one.d_k.stride_t = -1
    _refused(lib.lnx_attn_bwd(one, None), -4, b"workspace")
    one.d_v.stride_h = 65
    _refused(lib.lnx_attn_bwd(one, None), -2, b"aligned")


def test_attention_step_strides_of_single_elements():
    lib = _lib.load()

    def step(**kw):
        a = _lib.AttnStepArgs(**{**dict(B=1, H=4, Hkv=1, S=4096, d=64, dtype=_lib.LNX_BF16, scale=1.0), **kw})
        a.q, a.k, a.v = _lib.Tensor4(_ptr(), ODD, 64, 3), _lib.Tensor4(_ptr(), ODD, ODD, 3), _lib.Tensor4(_ptr(), ODD, ODD, 3)
        a.k_cache, a.v_cache = _lib.Tensor4(_ptr(), ODD, ODD, 64), _lib.Tensor4(_ptr(), ODD, ODD, 64)
        a.o = a.lengths = _ptr()
        return a

    _refused(lib.lnx_attn_step(step(), None), -4, b"workspace")
    _refused(lib.lnx_attn_step(step(B=2), None), -2, b"aligned")
    _refused(lib.lnx_attn_step(step(H=4, Hkv=2), None), -2, b"aligned")
    a = step()
    a.k_cache.stride_t = 65
    _refused(lib.lnx_attn_step(a, None), -2, b"aligned")


def test_recurrence_stride_of_a_single_token():
    lib = _lib.load()
    a = _lib.LinrecArgs(B=1 << 24, T=1, D=64, x_stride_t=1 << 40, g_stride_t=-1, d_y_stride_t=1 << 40)
    a.x = a.g = a.y = a.final_state = a.d_x = a.d_g = a.kept = _ptr()
    for fn in (lib.lnx_linrec_fwd, lib.lnx_linrec_bwd):
        _refused(fn(a, None), -2, b"too many rows")
    a.T = 2
    for fn in (lib.lnx_linrec_fwd, lib.lnx_linrec_bwd):
        _refused(fn(a, None), -2, b"apart")


def test_recorded_traffic_is_of_the_sources():
    """profiles/traffic.json is quoted only while the sources hash to what was measured.  Who changes one of them measures its kernels again or
    drops the entry; what only other kernels use belongs into a header of its own."""
    import bench

    with open(os.path.join(ROOT, "profiles", "traffic.json")) as f:
        entries = json.load(f)["measurements"]
    assert entries
    for e in entries:
        assert bench.sources_sha256(e["sources"]) == e["sources_sha256"], (e["commit"], e["sources"])
