"""ctypes binding of libhstu_rows8.so (the C ABI declared in include/hstu_rows8.h)."""

from __future__ import annotations

import ctypes as C
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("RECML_AMD_ROWS8_LIB") or os.path.join(_HERE, "lib", "libhstu_rows8.so")

ABI_VERSION = 1
BF16, FP32 = 0, 1
AS_IS, LAYER, RMS = 0, 1, 2
MAX_WIDTH = 32768

EXPORTS = (
    "hstu_rows8_abi_version",
    "hstu_rows8_last_error",
    "hstu_rows8_norm",
    "hstu_rows8_read",
    "hstu_rows8_gemm",
)


class HstuRows8(C.Structure):
  """Field-for-field image of `struct HstuRows8`."""

  _fields_ = [("codes", C.c_void_p), ("exponents", C.c_void_p), ("rows", C.c_int64), ("width", C.c_int32), ("reserved0", C.c_int32)]


class HstuRows8NormArgs(C.Structure):
  """Field-for-field image of `struct HstuRows8NormArgs`."""

  _fields_ = [
      ("struct_size", C.c_uint32), ("version", C.c_uint32),
      ("rows", HstuRows8), ("norm", C.c_int32), ("dtype", C.c_int32), ("eps", C.c_float), ("reserved0", C.c_int32),
      ("x", C.c_void_p), ("add", C.c_void_p), ("gate", C.c_void_p), ("sum", C.c_void_p),
      ("x_stride", C.c_int64), ("add_stride", C.c_int64), ("gate_stride", C.c_int64), ("sum_stride", C.c_int64),
      ("gamma", C.c_void_p), ("beta", C.c_void_p),
  ]


class HstuRows8ReadArgs(C.Structure):
  """Field-for-field image of `struct HstuRows8ReadArgs`."""

  _fields_ = [
      ("struct_size", C.c_uint32), ("version", C.c_uint32),
      ("rows", HstuRows8), ("out", C.c_void_p), ("out_stride", C.c_int64), ("dtype", C.c_int32), ("reserved0", C.c_int32),
  ]


class HstuRows8GemmArgs(C.Structure):
  """Field-for-field image of `struct HstuRows8GemmArgs`."""

  _fields_ = [
      ("struct_size", C.c_uint32), ("version", C.c_uint32),
      ("x", HstuRows8), ("w", HstuRows8), ("dtype", C.c_int32), ("activation", C.c_int32),
      ("out", C.c_void_p), ("c", C.c_void_p), ("bias", C.c_void_p), ("out_stride", C.c_int64), ("c_stride", C.c_int64),
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
    lib.hstu_rows8_abi_version.restype = C.c_int
    lib.hstu_rows8_abi_version.argtypes = []
    lib.hstu_rows8_last_error.restype = C.c_char_p
    lib.hstu_rows8_last_error.argtypes = []
    for name, args in (("hstu_rows8_norm", HstuRows8NormArgs), ("hstu_rows8_read", HstuRows8ReadArgs), ("hstu_rows8_gemm", HstuRows8GemmArgs)):
      fn = getattr(lib, name)
      fn.restype = C.c_int
      fn.argtypes = [C.POINTER(args), C.c_void_p]
    ver = lib.hstu_rows8_abi_version()
    if ver != ABI_VERSION:
      raise RuntimeError(f"libhstu_rows8.so has ABI {ver}, expected {ABI_VERSION}")
    _lib = lib
  return _lib
