"""ctypes binding of ``libpiper_b200.so`` (the C ABI declared in ``include/piper_b200.h``).

There is no fallback: if the shared library is missing or a call fails, an exception is
raised.  Build the library with ``python -m piper_kernels_b200.csrc.build``.
"""

from __future__ import annotations

import ctypes as C
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libpiper_b200.so"

PK_OK = 0
PK_ERR_BAD_ARG, PK_ERR_UNSUPPORTED_ARCH, PK_ERR_WORKSPACE, PK_ERR_CUDA, PK_ERR_DEVICE_STATUS = 1, 2, 3, 4, 5
PK_F16, PK_BF16, PK_F32, PK_I8 = 0, 1, 2, 3
PK_QK_PER_BLOCK, PK_QK_PER_THREAD = 0, 1
PK_CACHE_MAP_BYTES = 768

EXPORTS = (
    "pk_version", "pk_last_error",
    "pk_piper_workspace_bytes", "pk_piper_prepare", "pk_piper_run", "pk_piper_attention_fwd",
    "pk_sage2pp_workspace_bytes", "pk_sage2pp_prepare", "pk_sage2pp_run", "pk_sage2pp_attention_fwd",
    "pk_device_status", "pk_debug_first_tile", "pk_kv_means_static", "pk_debug_timeline",
    "pk_piper_prepare_kv", "pk_piper_prepare_q", "pk_sage2pp_prepare_kv", "pk_sage2pp_prepare_q",
    "pk_poll_device_fault", "pk_debug_stalled_wait",
    "pk_window_workspace_bytes", "pk_window_attention_fwd",
    "pk_cache_maps", "pk_cache_extend", "pk_cache_write", "pk_cache_read", "pk_cache_fork", "pk_cache_truncate", "pk_cache_compact",
    "pk_cache_attention_workspace_bytes", "pk_cache_attention_fwd", "pk_debug_window_stall", "pk_debug_cache_stall",
)


class PkProblem(C.Structure):
    _fields_ = [
        ("batch", C.c_int32), ("heads", C.c_int32), ("q_len", C.c_int32), ("kv_len", C.c_int32),
        ("head_dim", C.c_int32), ("in_dtype", C.c_int32), ("out_dtype", C.c_int32),
        ("is_causal", C.c_int32), ("center_value", C.c_int32), ("sort_value_rows", C.c_int32),
        ("qk_granularity", C.c_int32), ("scale", C.c_float),
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p),
        ("q_stride", C.c_int64 * 3), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3),
        ("out", C.c_void_p),
        ("k_mean_override", C.c_void_p), ("v_mean_override", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
        ("device", C.c_int32), ("stream", C.c_void_p),
    ]


class PkViews(C.Structure):
    _fields_ = [
        ("q_codes", C.c_void_p), ("k_codes", C.c_void_p), ("v_codes_t", C.c_void_p),
        ("q_group_scale", C.c_void_p), ("k_group_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("k_mean", C.c_void_p), ("v_mean", C.c_void_p), ("order", C.c_void_p),
        ("q_row_mul", C.c_void_p), ("k_col_mul", C.c_void_p), ("k_col_add", C.c_void_p),
        ("k_col_inv", C.c_void_p), ("status", C.c_void_p),
        ("sq_pad", C.c_int32), ("sk_pad", C.c_int32),
    ]


class PkWindowProblem(C.Structure):
    _fields_ = [
        ("batch", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32), ("q_len", C.c_int32),
        ("kv_len", C.c_int32), ("head_dim", C.c_int32), ("dtype", C.c_int32), ("window", C.c_int32),
        ("sinks", C.c_int32), ("scale", C.c_float),
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p),
        ("q_stride", C.c_int64 * 3), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3),
        ("lengths", C.c_void_p), ("out", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
        ("device", C.c_int32), ("stream", C.c_void_p),
    ]


class PkCache(C.Structure):
    _fields_ = [
        ("layers", C.c_int32), ("pages", C.c_int32), ("kv_heads", C.c_int32), ("page_size", C.c_int32),
        ("head_dim", C.c_int32), ("batch", C.c_int32), ("width", C.c_int32), ("dtype", C.c_int32),
        ("keys", C.c_void_p), ("values", C.c_void_p), ("key_scales", C.c_void_p), ("value_scales", C.c_void_p),
        ("table", C.c_void_p), ("lengths", C.c_void_p), ("starts", C.c_void_p), ("uses", C.c_void_p),
        ("refused", C.c_void_p), ("scratch", C.c_void_p), ("maps", C.c_void_p),
        ("device", C.c_int32), ("stream", C.c_void_p),
    ]


class PkCacheQuery(C.Structure):
    _fields_ = [
        ("heads", C.c_int32), ("tokens", C.c_int32), ("layer", C.c_int32), ("dtype", C.c_int32),
        ("window", C.c_int32), ("sinks", C.c_int32), ("scale", C.c_float),
        ("q", C.c_void_p), ("q_stride", C.c_int64 * 3), ("tree", C.c_void_p), ("tree_stride", C.c_int64),
        ("out", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
    ]


class PiperB200Error(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"libpiper_b200 error {code}: {message}")
        self.code = code


_lib = None


def lib() -> C.CDLL:
    """Load the shared library once; raise if it is absent (no fallback path exists)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m piper_kernels_b200.csrc.build` "
                "(needs nvcc with sm_100a support); piper_kernels_b200 has no other backend")
        handle = C.CDLL(str(LIB_PATH))
        P, V = C.POINTER(PkProblem), C.POINTER(PkViews)
        handle.pk_version.restype = C.c_int
        handle.pk_last_error.restype = C.c_char_p
        for name in ("pk_piper_workspace_bytes", "pk_sage2pp_workspace_bytes"):
            getattr(handle, name).argtypes = [P, C.POINTER(C.c_uint64)]
        for name in ("pk_piper_prepare", "pk_sage2pp_prepare", "pk_piper_prepare_kv", "pk_piper_prepare_q",
                     "pk_sage2pp_prepare_kv", "pk_sage2pp_prepare_q"):
            getattr(handle, name).argtypes = [P, V]
        for name in ("pk_piper_run", "pk_piper_attention_fwd", "pk_sage2pp_run", "pk_sage2pp_attention_fwd"):
            getattr(handle, name).argtypes = [P]
        handle.pk_device_status.argtypes = [P, C.POINTER(C.c_int32 * 16)]
        handle.pk_debug_first_tile.argtypes = [P, C.c_int, C.c_int, C.c_int, C.c_void_p]
        handle.pk_debug_timeline.argtypes = [P, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int]
        handle.pk_kv_means_static.argtypes = [P, C.c_void_p, C.c_void_p]
        handle.pk_poll_device_fault.argtypes = [C.c_int32, C.POINTER(C.c_int32)]
        handle.pk_debug_stalled_wait.argtypes = [P, C.c_int, C.c_int]
        W, K, Q = C.POINTER(PkWindowProblem), C.POINTER(PkCache), C.POINTER(PkCacheQuery)
        ptr, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
        handle.pk_window_workspace_bytes.argtypes = [W, C.POINTER(C.c_uint64)]
        handle.pk_window_attention_fwd.argtypes = [W]
        handle.pk_cache_maps.argtypes = [K, ptr]
        handle.pk_cache_extend.argtypes = [K, ptr]
        handle.pk_cache_write.argtypes = [K, i32, ptr, ptr, i64 * 4, i64 * 4, i32, i32]
        handle.pk_cache_read.argtypes = [K, i32, ptr, i32, ptr, ptr, i32]
        handle.pk_cache_fork.argtypes = [K, ptr]
        handle.pk_cache_truncate.argtypes = [K, ptr]
        handle.pk_cache_compact.argtypes = [K, ptr, i64, i32, ptr]
        handle.pk_cache_attention_workspace_bytes.argtypes = [K, Q, C.POINTER(C.c_uint64)]
        handle.pk_cache_attention_fwd.argtypes = [K, Q]
        handle.pk_debug_window_stall.argtypes = [W, i64, i32]
        handle.pk_debug_cache_stall.argtypes = [K, Q, i64, i32]
        for name in EXPORTS[2:]:
            getattr(handle, name).restype = C.c_int
        _lib = handle
    return _lib


def check(code: int) -> None:
    if code != PK_OK:
        raise PiperB200Error(code, lib().pk_last_error().decode("utf-8", "replace"))
