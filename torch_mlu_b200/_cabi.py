"""ctypes binding of libsdpa_b200.so (the C ABI declared in include/sdpa_b200.h).

The struct below mirrors ``sdpa_b200_params`` field for field. There is no fallback: if the
shared library is missing or a call returns a non-zero status, the caller gets an exception.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_char_p, c_float, c_int, c_int32, c_int64, c_size_t, c_uint64, c_void_p

LIB_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib")
LIB_PATH = os.path.join(LIB_DIR, "libsdpa_b200.so")

OK, INVALID_ARG, UNSUPPORTED, LAUNCH_FAILED, DEVICE_TIMEOUT, NO_DEVICE = range(6)
KERNEL_AUTO, KERNEL_PREFILL, KERNEL_DECODE = 0, 1, 2
DTYPE_BF16, DTYPE_F16 = 0, 1
CODE_E4M3, CODE_INT8, CODE_INT4 = 0, 1, 4

# every symbol include/sdpa_b200.h declares
EXPORTED_SYMBOLS = (
    "sdpa_b200_version",
    "sdpa_b200_status_string",
    "sdpa_b200_last_error",
    "sdpa_b200_fwd_workspace_bytes",
    "sdpa_b200_bwd_workspace_bytes",
    "sdpa_b200_bwd_workspace_least_bytes",
    "sdpa_b200_fwd",
    "sdpa_b200_bwd",
    "sdpa_b200_read_device_status",
    "sdpa_b200_selftest_wait_timeout",
    "sdpa_b200_selftest_grid_timeout",
    "sdpa_b200_decode_static",
    "sdpa_b200_merge_partial",
    "sdpa_b200_dropout_keep_mask",
    "sdpa_b200_dropout_keep_mask_varlen",
    "sdpa_b200_transpose_bias",
    "sdpa_b200_mask_to_bias",
    "sdpa_b200_pad_bias",
    "sdpa_b200_sum_bias_grad",
    "sdpa_b200_rotary",
    "sdpa_b200_plan_step",
    "sdpa_b200_cache_store",
    "sdpa_b200_cache_load",
    "sdpa_b200_cache_attention_workspace_bytes",
    "sdpa_b200_cache_attention",
    "sdpa_b200_launch_count",
)
STATIC_SCRATCH_BYTES = 16 << 20


class SdpaParams(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("k", c_void_p), ("v", c_void_p),
        ("out", c_void_p), ("lse", c_void_p),
        ("dout", c_void_p), ("dq", c_void_p), ("dk", c_void_p), ("dv", c_void_p),
        ("cu_seqlens_q", c_void_p), ("cu_seqlens_k", c_void_p),
        ("batch", c_int32), ("heads_q", c_int32), ("heads_kv", c_int32), ("head_dim", c_int32),
        ("max_seqlen_q", c_int32), ("max_seqlen_k", c_int32),
        ("total_q", c_int32), ("total_k", c_int32),
        ("q_batch_stride", c_int64), ("q_head_stride", c_int64), ("q_row_stride", c_int64),
        ("k_batch_stride", c_int64), ("k_head_stride", c_int64), ("k_row_stride", c_int64),
        ("v_batch_stride", c_int64), ("v_head_stride", c_int64), ("v_row_stride", c_int64),
        ("o_batch_stride", c_int64), ("o_head_stride", c_int64), ("o_row_stride", c_int64),
        ("do_batch_stride", c_int64), ("do_head_stride", c_int64), ("do_row_stride", c_int64),
        ("dq_batch_stride", c_int64), ("dq_head_stride", c_int64), ("dq_row_stride", c_int64),
        ("dk_batch_stride", c_int64), ("dk_head_stride", c_int64), ("dk_row_stride", c_int64),
        ("dv_batch_stride", c_int64), ("dv_head_stride", c_int64), ("dv_row_stride", c_int64),
        ("softmax_scale", c_float), ("dropout_p", c_float),
        ("is_causal", c_int32), ("dtype", c_int32), ("kernel", c_int32), ("num_splits", c_int32),
        ("keep_rows", c_void_p), ("keep_cols", c_void_p),
        ("bias", c_void_p), ("bias_batch_stride", c_int64), ("bias_head_stride", c_int64), ("bias_row_stride", c_int64),
        ("dbias", c_void_p), ("dbias_batch_stride", c_int64), ("dbias_head_stride", c_int64), ("dbias_row_stride", c_int64),
        ("bias_t", c_void_p), ("bias_t_batch_stride", c_int64), ("bias_t_head_stride", c_int64), ("bias_t_row_stride", c_int64),
        ("deterministic", c_int32), ("sm_margin", c_int32),
        ("device_status", c_void_p),
    ]


class RotaryParams(ctypes.Structure):
    _fields_ = [
        ("q", c_void_p), ("k", c_void_p), ("q_out", c_void_p), ("k_out", c_void_p),
        ("positions", c_void_p), ("inv_freq", c_void_p),
        ("batch", c_int32), ("length", c_int32), ("heads_q", c_int32), ("heads_k", c_int32),
        ("head_dim", c_int32), ("rotary_dim", c_int32), ("axes", c_int32), ("sections", c_int32 * 4),
        ("interleaved", c_int32), ("inverse", c_int32), ("positions_64", c_int32), ("dtype", c_int32), ("scaling", c_float),
        ("q_batch_stride", c_int64), ("q_head_stride", c_int64), ("q_row_stride", c_int64),
        ("k_batch_stride", c_int64), ("k_head_stride", c_int64), ("k_row_stride", c_int64),
        ("qo_batch_stride", c_int64), ("qo_head_stride", c_int64), ("qo_row_stride", c_int64),
        ("ko_batch_stride", c_int64), ("ko_head_stride", c_int64), ("ko_row_stride", c_int64),
        ("pos_axis_stride", c_int64), ("pos_batch_stride", c_int64), ("pos_row_stride", c_int64),
    ]


class PlanParams(ctypes.Structure):
    _fields_ = [
        ("cached_lens", c_void_p), ("new_tokens", c_void_p), ("block_table", c_void_p), ("ring", c_void_p), ("ring_state", c_void_p),
        ("seq_lens", c_void_p), ("cu_seqlens", c_void_p), ("positions", c_void_p), ("slots", c_void_p), ("next_state", c_void_p),
        ("table_stride", c_int64),
        ("batch", c_int32), ("max_blocks", c_int32), ("num_blocks", c_int32), ("block_size", c_int32), ("num_tokens", c_int32),
    ]


class CacheParams(ctypes.Structure):
    _fields_ = [
        ("k_cache", c_void_p), ("v_cache", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p),
        ("k_block_stride", c_int64), ("k_head_stride", c_int64), ("k_row_stride", c_int64),
        ("v_block_stride", c_int64), ("v_head_stride", c_int64), ("v_row_stride", c_int64),
        ("num_blocks", c_int32), ("block_size", c_int32), ("heads_kv", c_int32), ("head_dim", c_int32),
        ("code", c_int32), ("dtype", c_int32),
        ("key", c_void_p), ("value", c_void_p),
        ("key_row_stride", c_int64), ("key_head_stride", c_int64), ("value_row_stride", c_int64), ("value_head_stride", c_int64),
        ("slots", c_void_p), ("num_tokens", c_int32),
        ("batch", c_int32), ("q", c_void_p), ("out", c_void_p), ("lse", c_void_p),
        ("q_row_stride", c_int64), ("q_head_stride", c_int64), ("o_row_stride", c_int64), ("o_head_stride", c_int64),
        ("block_table", c_void_p), ("seq_lens", c_void_p), ("cu_seqlens_q", c_void_p), ("table_stride", c_int64),
        ("max_blocks", c_int32), ("heads_q", c_int32), ("total_q", c_int32), ("max_seqlen_q", c_int32), ("max_seqlen_k", c_int32),
        ("is_causal", c_int32), ("softmax_scale", c_float), ("device_status", c_void_p),
        ("key_out", c_void_p), ("value_out", c_void_p), ("first", c_void_p), ("cu_seqlens_k", c_void_p),
    ]


class SdpaError(RuntimeError):
    """A C-ABI call returned a non-zero status."""

    def __init__(self, status: int, text: str):
        super().__init__(text)
        self.status = status


_lib = None


def load() -> ctypes.CDLL:
    """dlopen the in-tree library; raise (never fall back) when it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m torch_mlu_b200.build` "
            "(there is no CPU or eager fallback for this path)"
        )
    lib = ctypes.CDLL(LIB_PATH)
    lib.sdpa_b200_version.restype = c_int
    lib.sdpa_b200_status_string.restype = c_char_p
    lib.sdpa_b200_status_string.argtypes = [c_int]
    lib.sdpa_b200_last_error.restype = c_char_p
    lib.sdpa_b200_launch_count.restype = c_uint64
    for name in ("sdpa_b200_fwd_workspace_bytes", "sdpa_b200_bwd_workspace_bytes", "sdpa_b200_bwd_workspace_least_bytes"):
        fn = getattr(lib, name)
        fn.restype = c_int
        fn.argtypes = [POINTER(SdpaParams), POINTER(c_size_t)]
    for name in ("sdpa_b200_fwd", "sdpa_b200_bwd"):
        fn = getattr(lib, name)
        fn.restype = c_int
        fn.argtypes = [POINTER(SdpaParams), c_void_p, c_size_t, c_void_p]
    lib.sdpa_b200_read_device_status.restype = c_int
    lib.sdpa_b200_read_device_status.argtypes = [c_void_p, c_void_p, POINTER(c_int)]
    lib.sdpa_b200_selftest_wait_timeout.restype = c_int
    lib.sdpa_b200_selftest_wait_timeout.argtypes = [c_void_p, ctypes.c_uint32, c_void_p]
    lib.sdpa_b200_selftest_grid_timeout.restype = c_int
    lib.sdpa_b200_selftest_grid_timeout.argtypes = [c_void_p, c_void_p, ctypes.c_uint32, ctypes.c_uint32, c_void_p]
    lib.sdpa_b200_decode_static.restype = c_int
    lib.sdpa_b200_decode_static.argtypes = [POINTER(SdpaParams), c_void_p]
    lib.sdpa_b200_merge_partial.restype = c_int
    lib.sdpa_b200_merge_partial.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32,
                                            c_int32, c_int64, c_int64, c_int64, c_void_p]
    lib.sdpa_b200_dropout_keep_mask.restype = c_int
    lib.sdpa_b200_dropout_keep_mask.argtypes = [c_uint64, c_uint64, c_float, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                c_void_p, c_void_p, c_void_p]
    lib.sdpa_b200_dropout_keep_mask_varlen.restype = c_int
    lib.sdpa_b200_dropout_keep_mask_varlen.argtypes = [c_uint64, c_uint64, c_float, c_int32, c_int32, c_void_p, c_void_p, c_int32,
                                                       c_int32, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p]
    lib.sdpa_b200_transpose_bias.restype = c_int
    lib.sdpa_b200_transpose_bias.argtypes = [c_void_p, c_int64, c_int64, c_int64, c_int32, c_int32, c_int32, c_int32, c_void_p,
                                             c_int64, c_void_p]
    lib.sdpa_b200_mask_to_bias.restype = c_int
    lib.sdpa_b200_mask_to_bias.argtypes = [c_void_p, c_int64, c_int64, c_int64, c_int64, c_int32, c_int32, c_int32, c_int32, c_void_p,
                                           c_int64, c_int32, c_void_p]
    lib.sdpa_b200_pad_bias.restype = c_int
    lib.sdpa_b200_pad_bias.argtypes = [c_void_p, c_int64, c_int64, c_int64, c_int64, c_int32, c_int32, c_int32, c_int32, c_void_p, c_int64,
                                       c_void_p]
    lib.sdpa_b200_sum_bias_grad.restype = c_int
    lib.sdpa_b200_sum_bias_grad.argtypes = [c_void_p, c_int64, c_int64, c_int64, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_void_p,
                                            c_int32, c_void_p]
    for name, struct in (("sdpa_b200_rotary", RotaryParams), ("sdpa_b200_plan_step", PlanParams), ("sdpa_b200_cache_store", CacheParams),
                         ("sdpa_b200_cache_load", CacheParams)):
        fn = getattr(lib, name)
        fn.restype = c_int
        fn.argtypes = [POINTER(struct), c_void_p]
    lib.sdpa_b200_cache_attention_workspace_bytes.restype = c_int
    lib.sdpa_b200_cache_attention_workspace_bytes.argtypes = [POINTER(CacheParams), POINTER(c_size_t)]
    lib.sdpa_b200_cache_attention.restype = c_int
    lib.sdpa_b200_cache_attention.argtypes = [POINTER(CacheParams), c_void_p, c_size_t, c_void_p]
    _lib = lib
    return lib


def check(status: int, what: str) -> None:
    if status != OK:
        lib = load()
        kind = lib.sdpa_b200_status_string(status).decode()
        detail = lib.sdpa_b200_last_error().decode()
        raise SdpaError(status, f"{what}: {kind}: {detail}")


def launch_count() -> int:
    return int(load().sdpa_b200_launch_count())
