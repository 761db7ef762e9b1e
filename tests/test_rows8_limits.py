"""Rows in 8 bits: calls of more threads than a launch has are refused as such (no GPU)."""

import ctypes as C

import pytest

from recml_amd import _lib_rows8


def _rows(r, rows, width):
  r.codes, r.exponents, r.rows, r.width = 0x10000, 0x20000, rows, width


@pytest.mark.parametrize("rows,width", [((1 << 29) + 32, 64), ((1 << 26) + 4, 512), ((1 << 22) + 1, 32768), ((1 << 31) - 1, 65)])
@pytest.mark.parametrize("norm", [_lib_rows8.AS_IS, _lib_rows8.LAYER])
def test_norm_of_too_many_rows(rows, width, norm):
  a = _lib_rows8.HstuRows8NormArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  _rows(a.rows, rows, width)
  a.norm, a.dtype, a.x, a.gamma, a.x_stride = norm, _lib_rows8.BF16, 0x3000, 0x4000, width
  lib = _lib_rows8.load()
  assert lib.hstu_rows8_norm(C.byref(a), None) == -4
  assert "too many" in lib.hstu_rows8_last_error().decode()


@pytest.mark.parametrize("dtype", [_lib_rows8.BF16, _lib_rows8.FP32])
@pytest.mark.parametrize("rows", [1, 16])
def test_product_of_few_rows_with_too_many_columns(rows, dtype):
  """Sixteen columns a workgroup of 512 threads."""
  a = _lib_rows8.HstuRows8GemmArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  _rows(a.x, rows, 2048)
  _rows(a.w, (1 << 27) + 16, 2048)
  a.out, a.out_stride, a.dtype = 0x3000, a.w.rows, dtype
  lib = _lib_rows8.load()
  assert lib.hstu_rows8_gemm(C.byref(a), None) == -4
  assert "too many" in lib.hstu_rows8_last_error().decode()
