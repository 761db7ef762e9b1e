"""ctypes binding of libhstu_serve.so (the C ABI declared in include/hstu_serve.h)."""

from __future__ import annotations

import ctypes as C
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("RECML_AMD_SERVE_LIB") or os.path.join(_HERE, "lib", "libhstu_serve.so")

ABI_VERSION = 1
BF16, FP32 = 0, 1

EXPORTS = (
    "hstu_serve_abi_version",
    "hstu_serve_last_error",
    "hstu_kv_write",
    "hstu_kv_read",
    "hstu_cached_attn",
    "hstu_cached_attn_workspace_bytes",
    "hstu_log_probs_fwd",
    "hstu_log_probs_bwd",
    "hstu_log_probs_workspace_bytes",
)


class HstuKvPages(C.Structure):
  """Field-for-field image of `struct HstuKvPages`."""

  _fields_ = [
      ("k_codes", C.c_void_p), ("k_scales", C.c_void_p), ("v_codes", C.c_void_p), ("v_scales", C.c_void_p),
      ("page_table", C.c_void_p),
      ("n_pages", C.c_int32), ("page_size", C.c_int32), ("table_pages", C.c_int32),
      ("B", C.c_int32), ("H", C.c_int32), ("d", C.c_int32), ("bits", C.c_int32), ("reserved0", C.c_int32),
  ]


class HstuKvRowsArgs(C.Structure):
  """Field-for-field image of `struct HstuKvRowsArgs`."""

  _fields_ = [
      ("struct_size", C.c_uint32), ("version", C.c_uint32),
      ("pages", HstuKvPages), ("starts", C.c_void_p), ("offsets", C.c_void_p),
      ("total_rows", C.c_int64), ("rows_per_seq", C.c_int32), ("dtype", C.c_int32),
      ("k", C.c_void_p), ("v", C.c_void_p),
      ("k_stride_b", C.c_int64), ("k_stride_t", C.c_int64), ("k_stride_h", C.c_int64),
      ("v_stride_b", C.c_int64), ("v_stride_t", C.c_int64), ("v_stride_h", C.c_int64),
  ]


class HstuCachedAttnArgs(C.Structure):
  """Field-for-field image of `struct HstuCachedAttnArgs`."""

  _fields_ = [
      ("struct_size", C.c_uint32), ("version", C.c_uint32),
      ("pages", HstuKvPages), ("lengths", C.c_void_p), ("offsets", C.c_void_p),
      ("total_rows", C.c_int64), ("rows_per_seq", C.c_int32), ("dtype", C.c_int32),
      ("q", C.c_void_p), ("out", C.c_void_p),
      ("q_stride_b", C.c_int64), ("q_stride_t", C.c_int64), ("q_stride_h", C.c_int64),
      ("o_stride_b", C.c_int64), ("o_stride_t", C.c_int64), ("o_stride_h", C.c_int64),
      ("max_len", C.c_int32), ("alpha", C.c_float), ("inv_n", C.c_float), ("pos_heads", C.c_int32),
      ("pos_tab", C.c_void_p), ("timestamps", C.c_void_p), ("ts_tab", C.c_void_p),
      ("ts_heads", C.c_int32), ("ts_buckets", C.c_int32), ("ts_bucket_size", C.c_float), ("reserved0", C.c_int32),
      ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
  ]


class HstuLogProbsArgs(C.Structure):
  """Field-for-field image of `struct HstuLogProbsArgs`."""

  _fields_ = [
      ("struct_size", C.c_uint32), ("version", C.c_uint32),
      ("logits", C.c_void_p), ("rows", C.c_int64), ("stride", C.c_int64),
      ("vocab", C.c_int32), ("dtype", C.c_int32), ("count", C.c_int32), ("top", C.c_int32),
      ("tokens", C.c_void_p), ("log_probs", C.c_void_p), ("entropy", C.c_void_p), ("stats", C.c_void_p),
      ("top_log_probs", C.c_void_p), ("top_tokens", C.c_void_p),
      ("g_tokens", C.c_void_p), ("g_entropy", C.c_void_p), ("g_top", C.c_void_p),
      ("d_logits", C.c_void_p), ("d_stride", C.c_int64),
      ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
  ]


_lock = threading.Lock()
_lib = None


def load():
  """Loads the shared library; raises if it has not been built (there is no fallback in here)."""
  global _lib
  if _lib is not None:
    return _lib
  with _lock:
    if _lib is not None:
      return _lib
    if not os.path.exists(LIB_PATH):
      raise RuntimeError(
          f"{LIB_PATH} is missing: build it with `python -m recml_amd.build` (needs hipcc)")
    lib = C.CDLL(LIB_PATH)
    lib.hstu_serve_abi_version.restype = C.c_int
    lib.hstu_serve_abi_version.argtypes = []
    lib.hstu_serve_last_error.restype = C.c_char_p
    lib.hstu_serve_last_error.argtypes = []
    for name, args in (("hstu_kv_write", HstuKvRowsArgs), ("hstu_kv_read", HstuKvRowsArgs), ("hstu_cached_attn", HstuCachedAttnArgs),
                       ("hstu_log_probs_fwd", HstuLogProbsArgs), ("hstu_log_probs_bwd", HstuLogProbsArgs)):
      fn = getattr(lib, name)
      fn.restype = C.c_int
      fn.argtypes = [C.POINTER(args), C.c_void_p]
    for name, args in (("hstu_cached_attn_workspace_bytes", HstuCachedAttnArgs), ("hstu_log_probs_workspace_bytes", HstuLogProbsArgs)):
      fn = getattr(lib, name)
      fn.restype = C.c_size_t
      fn.argtypes = [C.POINTER(args)]
    ver = lib.hstu_serve_abi_version()
    if ver != ABI_VERSION:
      raise RuntimeError(f"libhstu_serve.so has ABI {ver}, expected {ABI_VERSION}")
    _lib = lib
  return _lib
