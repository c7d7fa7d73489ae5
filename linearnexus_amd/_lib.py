"""ctypes binding of liblinearnexus_hip.so (the C-ABI declared in include/linearnexus_hip.h).

There is no fallback: if the library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "liblinearnexus_hip.so")

LNX_F32, LNX_BF16 = 0, 1
STATIC_SCRATCH_BYTES = 64 << 20  # LNX_STATIC_SCRATCH_BYTES
GATE_NONE, GATE_SCALAR, GATE_VECTOR = 0, 1, 2

EXPORTS = (
    "lnx_abi_version", "lnx_last_error", "lnx_decode_step", "lnx_recurrent_fwd",
    "lnx_chunk_workspace_bytes", "lnx_chunk_normalises_qk", "lnx_chunk_fuses_l2norm", "lnx_chunk_fwd", "lnx_chunk_fwd_segmented_bytes", "lnx_chunk_fwd_segmented", "lnx_chunk_fwd_segmented_final", "lnx_chunk_fwd_static", "lnx_chunk_fwd_static_init", "lnx_chunk_bwd", "lnx_chunk_bwd_d_o32", "lnx_chunk_rounds_d_o", "lnx_l2norm_fwd", "lnx_l2norm_bwd", "lnx_l2norm_pair_fwd", "lnx_l2norm_pair_bwd",
    "lnx_conv1d_fwd", "lnx_conv1d_bwd", "lnx_conv1d_cache_bwd", "lnx_conv1d_packed_fwd", "lnx_conv1d_packed_bwd", "lnx_conv1d_fwd_zero", "lnx_conv1d_bwd_add", "lnx_dplr_recurrent_fwd", "lnx_dplr_step", "lnx_dplr_recurrent_bwd", "lnx_dplr_recurrent_bwd_workspace_bytes", "lnx_dplr_chunk_fits", "lnx_dplr_chunk_bytes", "lnx_dplr_chunk_fwd", "lnx_dplr_chunk_bwd", "lnx_rmsnorm_gated_fwd", "lnx_rmsnorm_gated_bwd", "lnx_rmsnorm_gated_bwd_workspace_bytes",
    "lnx_gdn_gate_fwd", "lnx_gdn_gate_bwd", "lnx_gdn_gate_bwd_workspace_bytes", "lnx_kda_gate_fwd", "lnx_kda_gate_bwd", "lnx_kda_gate_bwd_workspace_bytes", "lnx_sigmoid_fwd", "lnx_sigmoid_bwd",
    "lnx_linrec_workspace_bytes", "lnx_linrec_kept_bytes", "lnx_linrec_fwd", "lnx_linrec_bwd", "lnx_linrec_step",
    "lnx_rmsnorm_residual_bwd_workspace_bytes", "lnx_rmsnorm_residual_fwd", "lnx_rmsnorm_residual_bwd",
    "lnx_layer_norm_bwd_workspace_bytes", "lnx_layer_norm_fwd", "lnx_layer_norm_bwd",
    "lnx_attn_fwd_workspace_bytes", "lnx_attn_bwd_workspace_bytes", "lnx_attn_fwd", "lnx_attn_bwd", "lnx_attn_step_workspace_bytes", "lnx_attn_step", "lnx_attn_step_paged_workspace_bytes", "lnx_attn_step_paged",
    "lnx_decay_kept_bytes", "lnx_decay_fwd_workspace_bytes", "lnx_decay_bwd_workspace_bytes", "lnx_decay_fwd", "lnx_decay_bwd", "lnx_decay_step",
    "lnx_profile_enable", "lnx_profile_read",
)


class ScanArgs(C.Structure):
    """Mirror of ``struct lnx_scan_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("T", C.c_int32), ("dk", C.c_int32), ("dv", C.c_int32),
        ("chunk", C.c_int32), ("dtype", C.c_int32), ("o_dtype", C.c_int32), ("gate", C.c_int32),
        ("use_qk_l2norm", C.c_int32), ("nseq", C.c_int32), ("scale", C.c_float),
        ("forward_only", C.c_int32), ("token_first", C.c_int32),
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("beta", C.c_void_p), ("g", C.c_void_p),
        ("initial_state", C.c_void_p), ("cu_seqlens", C.c_void_p), ("o", C.c_void_p),
        ("final_state", C.c_void_p),
        ("d_o", C.c_void_p), ("d_final_state", C.c_void_p), ("d_q", C.c_void_p), ("d_k", C.c_void_p),
        ("d_v", C.c_void_p), ("d_beta", C.c_void_p), ("d_g", C.c_void_p), ("d_initial_state", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
        ("value_cols", C.c_int32),
        ("gate_raw", C.c_void_p), ("gate_A_log", C.c_void_p), ("gate_bias", C.c_void_p), ("gate_threshold", C.c_float),
        ("d_gate_raw", C.c_void_p), ("d_gate_A_log", C.c_void_p), ("d_gate_bias", C.c_void_p),
        ("test_scan_slab", C.c_int32), ("test_out_slabs", C.c_int32),
    ]


class DplrArgs(C.Structure):
    """Mirror of ``struct lnx_dplr_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("T", C.c_int32), ("dk", C.c_int32), ("dv", C.c_int32),
        ("dtype", C.c_int32), ("o_dtype", C.c_int32), ("scale", C.c_float),
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("a", C.c_void_p), ("b", C.c_void_p),
        ("gk", C.c_void_p), ("initial_state", C.c_void_p), ("o", C.c_void_p), ("final_state", C.c_void_p),
    ]


class DplrBwdArgs(C.Structure):
    """Mirror of ``struct lnx_dplr_bwd_args``."""

    _fields_ = [
        ("fwd", DplrArgs), ("d_o", C.c_void_p), ("d_final_state", C.c_void_p),
        ("dq", C.c_void_p), ("dk", C.c_void_p), ("dv", C.c_void_p), ("da", C.c_void_p), ("db", C.c_void_p),
        ("dgk", C.c_void_p), ("d_initial_state", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class LinrecArgs(C.Structure):
    """Mirror of ``struct lnx_linrec_args``."""

    _fields_ = [
        ("B", C.c_int32), ("T", C.c_int32), ("D", C.c_int32), ("nseq", C.c_int32), ("dtype", C.c_int32), ("g_dtype", C.c_int32),
        ("x_stride_b", C.c_int64), ("x_stride_t", C.c_int64), ("g_stride_b", C.c_int64), ("g_stride_t", C.c_int64),
        ("d_y_stride_b", C.c_int64), ("d_y_stride_t", C.c_int64),
        ("x", C.c_void_p), ("g", C.c_void_p), ("initial_state", C.c_void_p), ("cu_seqlens", C.c_void_p), ("y", C.c_void_p),
        ("final_state", C.c_void_p), ("kept", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
        ("d_y", C.c_void_p), ("d_final_state", C.c_void_p), ("d_x", C.c_void_p), ("d_g", C.c_void_p), ("d_initial_state", C.c_void_p),
    ]


class RmsnormResidualArgs(C.Structure):
    """Mirror of ``struct lnx_rmsnorm_residual_args``."""

    _fields_ = [
        ("rows", C.c_int64), ("d", C.c_int32), ("dtype", C.c_int32), ("r_dtype", C.c_int32), ("scale", C.c_float), ("eps", C.c_float),
        ("gate_f32", C.c_int32),
        ("x", C.c_void_p), ("residual", C.c_void_p), ("gate", C.c_void_p), ("weight", C.c_void_p), ("post_weight", C.c_void_p),
        ("scale_vector", C.c_void_p), ("z", C.c_void_p), ("out", C.c_void_p), ("d_z", C.c_void_p), ("d_out", C.c_void_p), ("d_x", C.c_void_p),
        ("d_residual", C.c_void_p), ("d_gate", C.c_void_p), ("d_weight", C.c_void_p), ("d_post_weight", C.c_void_p), ("d_scale", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class LayerNormArgs(C.Structure):
    """Mirror of ``struct lnx_layer_norm_args``."""

    _fields_ = [
        ("rows", C.c_int64), ("heads", C.c_int32), ("d", C.c_int32), ("dtype", C.c_int32), ("eps", C.c_float),
        ("x", C.c_void_p), ("weight", C.c_void_p), ("bias", C.c_void_p), ("y", C.c_void_p), ("d_y", C.c_void_p), ("d_x", C.c_void_p),
        ("d_weight", C.c_void_p), ("d_bias", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class Tensor4(C.Structure):
    """Mirror of ``struct lnx_tensor4``."""

    _fields_ = [("p", C.c_void_p), ("stride_b", C.c_int64), ("stride_h", C.c_int64), ("stride_t", C.c_int64)]


class AttnArgs(C.Structure):
    """Mirror of ``struct lnx_attn_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("T", C.c_int32), ("d", C.c_int32), ("nseq", C.c_int32), ("dtype", C.c_int32),
        ("scale", C.c_float),
        ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("o", Tensor4), ("d_o", Tensor4), ("d_q", Tensor4), ("d_k", Tensor4), ("d_v", Tensor4),
        ("lse", C.c_void_p), ("o_low", C.c_void_p), ("cu_seqlens", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class AttnStepArgs(C.Structure):
    """Mirror of ``struct lnx_attn_step_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("S", C.c_int32), ("d", C.c_int32), ("dtype", C.c_int32),
        ("scale", C.c_float), ("reserved", C.c_int32),
        ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("k_cache", Tensor4), ("v_cache", Tensor4),
        ("o", C.c_void_p), ("lengths", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class AttnStepPagedArgs(C.Structure):
    """Mirror of ``struct lnx_attn_step_paged_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("Hkv", C.c_int32), ("d", C.c_int32), ("dtype", C.c_int32),
        ("page", C.c_int32), ("pages", C.c_int32), ("table_width", C.c_int32), ("scale", C.c_float), ("reserved", C.c_int32),
        ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("k_cache", Tensor4), ("v_cache", Tensor4),
        ("o", C.c_void_p), ("lengths", C.c_void_p), ("page_table", C.c_void_p), ("table_stride", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class DecayArgs(C.Structure):
    """Mirror of ``struct lnx_decay_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("T", C.c_int32), ("dk", C.c_int32), ("dv", C.c_int32), ("nseq", C.c_int32), ("dtype", C.c_int32),
        ("g_per_head", C.c_int32), ("scale", C.c_float), ("reserved", C.c_int32),
        ("q", Tensor4), ("k", Tensor4), ("v", Tensor4), ("o", Tensor4), ("d_o", Tensor4), ("d_q", Tensor4), ("d_k", Tensor4), ("d_v", Tensor4),
        ("g", C.c_void_p), ("g_stride_b", C.c_int64), ("g_stride_h", C.c_int64), ("g_stride_t", C.c_int64), ("cu_seqlens", C.c_void_p),
        ("initial_state", C.c_void_p), ("final_state", C.c_void_p), ("kept", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
        ("d_final_state", C.c_void_p), ("d_g", C.c_void_p), ("d_initial_state", C.c_void_p),
    ]


class DecayStepArgs(C.Structure):
    """Mirror of ``struct lnx_decay_step_args``."""

    _fields_ = [
        ("B", C.c_int32), ("H", C.c_int32), ("dk", C.c_int32), ("dv", C.c_int32), ("dtype", C.c_int32), ("scale", C.c_float),
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("g", C.c_void_p), ("g_stride_b", C.c_int64), ("g_stride_h", C.c_int64),
        ("state", C.c_void_p), ("o", C.c_void_p), ("new_state", C.c_void_p),
    ]


_lib = None


def load() -> C.CDLL:
    """Loads the library once; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m linearnexus_amd.build` "
            "(there is no CPU or PyTorch fallback for these ops)"
        )
    lib = C.CDLL(LIB_PATH)
    lib.lnx_abi_version.restype = C.c_int
    lib.lnx_last_error.restype = C.c_char_p
    for name in ("lnx_decode_step", "lnx_recurrent_fwd", "lnx_chunk_fwd", "lnx_chunk_fwd_static", "lnx_chunk_bwd"):
        fn = getattr(lib, name)
        fn.restype = C.c_int
        fn.argtypes = [C.POINTER(ScanArgs), C.c_void_p]
    lib.lnx_chunk_bwd_d_o32.restype = C.c_int
    lib.lnx_chunk_bwd_d_o32.argtypes = [C.POINTER(ScanArgs), C.c_void_p, C.c_void_p]
    lib.lnx_chunk_fwd_static_init.restype = C.c_int
    lib.lnx_chunk_fwd_static_init.argtypes = []
    lib.lnx_chunk_workspace_bytes.restype = C.c_uint64
    lib.lnx_chunk_workspace_bytes.argtypes = [C.POINTER(ScanArgs)]
    for name in ("lnx_chunk_normalises_qk", "lnx_chunk_fuses_l2norm", "lnx_chunk_rounds_d_o"):
        getattr(lib, name).restype = C.c_int
        getattr(lib, name).argtypes = [C.POINTER(ScanArgs)]
    lib.lnx_l2norm_fwd.restype = C.c_int
    lib.lnx_l2norm_fwd.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int32, C.c_int32, C.c_void_p]
    lib.lnx_l2norm_bwd.restype = C.c_int
    lib.lnx_l2norm_bwd.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int32, C.c_int32, C.c_void_p]
    lib.lnx_conv1d_fwd.restype = C.c_int
    lib.lnx_conv1d_fwd.argtypes = [C.c_void_p] * 6 + [C.c_int32] * 6 + [C.c_void_p]
    lib.lnx_conv1d_bwd.restype = C.c_int
    lib.lnx_conv1d_bwd.argtypes = [C.c_void_p] * 8 + [C.c_int32] * 6 + [C.c_void_p]
    lib.lnx_conv1d_cache_bwd.restype = C.c_int
    lib.lnx_conv1d_cache_bwd.argtypes = [C.c_void_p] * 6 + [C.c_int32] * 6 + [C.c_void_p]
    lib.lnx_conv1d_packed_fwd.restype = C.c_int
    lib.lnx_conv1d_packed_fwd.argtypes = [C.c_void_p] * 4 + [C.c_int32] + [C.c_void_p] * 2 + [C.c_int32] * 5 + [C.c_void_p]
    lib.lnx_conv1d_packed_bwd.restype = C.c_int
    lib.lnx_conv1d_packed_bwd.argtypes = [C.c_void_p] * 4 + [C.c_int32] + [C.c_void_p] * 4 + [C.c_int32] * 5 + [C.c_void_p]
    lib.lnx_rmsnorm_gated_fwd.restype = C.c_int
    lib.lnx_rmsnorm_gated_fwd.argtypes = [C.c_void_p] * 4 + [C.c_int64, C.c_int32, C.c_float, C.c_int32, C.c_void_p]
    lib.lnx_rmsnorm_gated_bwd.restype = C.c_int
    lib.lnx_rmsnorm_gated_bwd.argtypes = [C.c_void_p] * 7 + [C.c_int64, C.c_int32, C.c_float, C.c_int32, C.c_void_p, C.c_uint64,
                                          C.c_void_p]
    lib.lnx_rmsnorm_gated_bwd_workspace_bytes.restype = C.c_uint64
    lib.lnx_rmsnorm_gated_bwd_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32]
    lib.lnx_kda_gate_fwd.restype = C.c_int
    lib.lnx_kda_gate_fwd.argtypes = [C.c_void_p] * 4 + [C.c_int64, C.c_int32, C.c_int32, C.c_float, C.c_int32, C.c_int32, C.c_void_p]
    lib.lnx_kda_gate_bwd_workspace_bytes.restype = C.c_uint64
    lib.lnx_kda_gate_bwd_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32]
    lib.lnx_kda_gate_bwd.restype = C.c_int
    lib.lnx_kda_gate_bwd.argtypes = [C.c_void_p] * 7 + [C.c_int64, C.c_int32, C.c_int32, C.c_float, C.c_int32, C.c_int32,
                                                         C.c_void_p, C.c_uint64, C.c_void_p]
    lib.lnx_gdn_gate_fwd.restype = C.c_int
    lib.lnx_gdn_gate_fwd.argtypes = [C.c_void_p] * 6 + [C.c_int64, C.c_int32, C.c_float, C.c_int32, C.c_void_p]
    lib.lnx_gdn_gate_bwd_workspace_bytes.restype = C.c_uint64
    lib.lnx_gdn_gate_bwd_workspace_bytes.argtypes = [C.c_int64, C.c_int32]
    lib.lnx_gdn_gate_bwd.restype = C.c_int
    lib.lnx_gdn_gate_bwd.argtypes = [C.c_void_p] * 10 + [C.c_int64, C.c_int32, C.c_float, C.c_int32, C.c_void_p, C.c_uint64, C.c_void_p]
    lib.lnx_sigmoid_fwd.restype = C.c_int
    lib.lnx_sigmoid_fwd.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    lib.lnx_sigmoid_bwd.restype = C.c_int
    lib.lnx_sigmoid_bwd.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    for name in ("lnx_dplr_recurrent_fwd", "lnx_dplr_step"):
        fn = getattr(lib, name)
        fn.restype = C.c_int
        fn.argtypes = [C.POINTER(DplrArgs), C.c_void_p]
    lib.lnx_dplr_recurrent_bwd.restype = C.c_int
    lib.lnx_dplr_recurrent_bwd.argtypes = [C.POINTER(DplrBwdArgs), C.c_void_p]
    lib.lnx_dplr_recurrent_bwd_workspace_bytes.restype = C.c_uint64
    lib.lnx_dplr_recurrent_bwd_workspace_bytes.argtypes = [C.c_int32] * 5
    for name in ("lnx_linrec_workspace_bytes", "lnx_linrec_kept_bytes"):
        getattr(lib, name).restype = C.c_uint64
        getattr(lib, name).argtypes = [C.POINTER(LinrecArgs)]
    for name in ("lnx_linrec_fwd", "lnx_linrec_bwd"):
        getattr(lib, name).restype = C.c_int
        getattr(lib, name).argtypes = [C.POINTER(LinrecArgs), C.c_void_p]
    lib.lnx_linrec_step.restype = C.c_int
    lib.lnx_linrec_step.argtypes = [C.c_void_p] * 5 + [C.c_int64, C.c_int32, C.c_int32, C.c_void_p]
    lib.lnx_rmsnorm_residual_bwd_workspace_bytes.restype = C.c_uint64
    lib.lnx_rmsnorm_residual_bwd_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32]
    for name in ("lnx_rmsnorm_residual_fwd", "lnx_rmsnorm_residual_bwd"):
        getattr(lib, name).restype = C.c_int
        getattr(lib, name).argtypes = [C.POINTER(RmsnormResidualArgs), C.c_void_p]
    lib.lnx_layer_norm_bwd_workspace_bytes.restype = C.c_uint64
    lib.lnx_layer_norm_bwd_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32, C.c_int32]
    for name in ("lnx_layer_norm_fwd", "lnx_layer_norm_bwd"):
        getattr(lib, name).restype = C.c_int
        getattr(lib, name).argtypes = [C.POINTER(LayerNormArgs), C.c_void_p]
    for name in ("lnx_attn_fwd_workspace_bytes", "lnx_attn_bwd_workspace_bytes"):
        getattr(lib, name).restype = C.c_uint64
        getattr(lib, name).argtypes = [C.POINTER(AttnArgs)]
    for name in ("lnx_attn_fwd", "lnx_attn_bwd"):
        getattr(lib, name).restype = C.c_int
        getattr(lib, name).argtypes = [C.POINTER(AttnArgs), C.c_void_p]
    lib.lnx_attn_step_workspace_bytes.restype = C.c_uint64
    lib.lnx_attn_step_workspace_bytes.argtypes = [C.POINTER(AttnStepArgs)]
    lib.lnx_attn_step.restype = C.c_int
    lib.lnx_attn_step.argtypes = [C.POINTER(AttnStepArgs), C.c_void_p]
    lib.lnx_attn_step_paged_workspace_bytes.restype = C.c_uint64
    lib.lnx_attn_step_paged_workspace_bytes.argtypes = [C.POINTER(AttnStepPagedArgs)]
    lib.lnx_attn_step_paged.restype = C.c_int
    lib.lnx_attn_step_paged.argtypes = [C.POINTER(AttnStepPagedArgs), C.c_void_p]
    for name in ("lnx_decay_kept_bytes", "lnx_decay_fwd_workspace_bytes", "lnx_decay_bwd_workspace_bytes"):
        getattr(lib, name).restype = C.c_uint64
        getattr(lib, name).argtypes = [C.POINTER(DecayArgs)]
    for name in ("lnx_decay_fwd", "lnx_decay_bwd"):
        getattr(lib, name).restype = C.c_int
        getattr(lib, name).argtypes = [C.POINTER(DecayArgs), C.c_void_p]
    lib.lnx_decay_step.restype = C.c_int
    lib.lnx_decay_step.argtypes = [C.POINTER(DecayStepArgs), C.c_void_p]
    lib.lnx_profile_enable.restype = C.c_int
    lib.lnx_profile_enable.argtypes = [C.c_int]
    lib.lnx_profile_read.restype = C.c_int
    lib.lnx_profile_read.argtypes = [C.c_int, C.POINTER(C.c_char_p), C.POINTER(C.c_float)]
    _lib = lib
    return lib


class HipKernelError(RuntimeError):
    """A C-ABI call returned a negative status."""


_host = None


def host():
    """The native host path of the ops (csrc/host_ops.cpp); raises if it has not been built."""
    global _host
    if _host is None:
        load()
        try:
            from . import _host as module
        except ImportError as e:
            raise RuntimeError("linearnexus_amd/_host.so is missing or does not load: build it with `python -m linearnexus_amd.build` "
                               "(there is no CPU or PyTorch fallback for these ops)") from e
        module.set_kernel_error(HipKernelError)
        _host = module
    return _host


def profile_enable(on: bool) -> None:
    """Turns per-kernel HIP-event timing on or off for the calling thread."""
    load().lnx_profile_enable(int(on))


def profile_read(capacity: int = 8192):
    """Returns [(kernel name, milliseconds), ...] for the kernels launched since the last read."""
    names = (C.c_char_p * capacity)()
    ms = (C.c_float * capacity)()
    n = load().lnx_profile_read(capacity, names, ms)
    return [(names[i].decode(), float(ms[i])) for i in range(min(n, capacity))]


def check(status: int, what: str) -> None:
    if status != 0:
        msg = load().lnx_last_error().decode("utf-8", "replace")
        raise HipKernelError(f"{what} failed (status {status}): {msg}")
