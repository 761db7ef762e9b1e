"""What the entry points on rows in 8 bits refuse, before any work, and their ABI (no GPU)."""

import copy
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

import recml_amd
from recml_amd import _lib_rows8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _fill(r, rows=4, width=256):
  r.codes, r.exponents, r.rows, r.width = 0x10000, 0x20000, rows, width


def _norm_args(**kw):
  a = _lib_rows8.HstuRows8NormArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  _fill(a.rows)
  a.norm, a.dtype, a.eps, a.x, a.gamma, a.x_stride = _lib_rows8.LAYER, _lib_rows8.BF16, 1e-6, 0x3000, 0x4000, 256
  return _set(a, a.rows, kw)


def _read_args(**kw):
  a = _lib_rows8.HstuRows8ReadArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  _fill(a.rows)
  a.out, a.out_stride, a.dtype = 0x3000, 256, _lib_rows8.FP32
  return _set(a, a.rows, kw)


def _gemm_args(**kw):
  a = _lib_rows8.HstuRows8GemmArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  _fill(a.x)
  _fill(a.w, rows=64)
  a.out, a.out_stride, a.dtype = 0x3000, 64, _lib_rows8.BF16
  return _set(a, a.x, kw)


def _set(a, rows, kw):
  for name, value in kw.items():
    if name == "rows" or not hasattr(a, name):
      setattr(rows, name, value)
    else:
      setattr(a, name, value)
  return a


ROWS = [(dict(struct_size=8), -2, "struct_size"), (dict(version=99), -2, "version"), (dict(rows=-1), -4, "rows"), (dict(rows=1 << 31), -4, "rows"), (dict(width=0), -4, "width"),
        (dict(width=32769), -4, "width"), (dict(codes=None), -1, "null"), (dict(exponents=None), -1, "null"), (dict(codes=0x10008), -4, "16-byte"), (dict(exponents=0x20002), -4, "4-byte"),
        (dict(dtype=2), -4, "dtype")]


def _refused(fn, args, status, word):
  assert fn(C.byref(args), None) == status
  assert word in _lib_rows8.load().hstu_rows8_last_error().decode()


@pytest.mark.parametrize("change,status,word", ROWS + [
    (dict(x=None), -1, "x is null"), (dict(gamma=None), -1, "gamma"), (dict(norm=3), -4, "norm"), (dict(sum=0x5000), -4, "sum"), (dict(norm=0, gate=0x5000), -4, "no gate"), (dict(norm=0, add=0x5000), -4, "nothing added"), (dict(x=0x3001), -4, "aligned"),
    (dict(beta=0x4001), -4, "aligned"), (dict(rows=1 << 30), -4, "too many")])
def test_norm_refused(change, status, word):
  _refused(_lib_rows8.load().hstu_rows8_norm, _norm_args(**change), status, word)


@pytest.mark.parametrize("change,status,word", ROWS + [(dict(out=None), -1, "out is null"), (dict(out=0x3002), -4, "aligned"), (dict(rows=1 << 30), -4, "too many")])
def test_read_refused(change, status, word):
  _refused(_lib_rows8.load().hstu_rows8_read, _read_args(**change), status, word)


@pytest.mark.parametrize("change,status,word", ROWS + [
    (dict(out=None), -1, "out is null"), (dict(out=0x3001), -4, "aligned"), (dict(c=0x3001), -4, "aligned"), (dict(activation=2), -4, "activation"),
    (dict(rows=(1 << 31) - 1), -4, "too many")])
def test_gemm_refused(change, status, word):
  _refused(_lib_rows8.load().hstu_rows8_gemm, _gemm_args(**change), status, word)


def test_gemm_of_two_widths_and_too_many_columns_refused():
  lib = _lib_rows8.load()
  a = _gemm_args()
  a.w.width = 128
  _refused(lib.hstu_rows8_gemm, a, -4, "rows of 256")
  a = _gemm_args(rows=1 << 30)
  a.w.rows = 1 << 30
  _refused(lib.hstu_rows8_gemm, a, -4, "too many")


def test_null_and_nothing_to_do():
  lib = _lib_rows8.load()
  for fn in (lib.hstu_rows8_norm, lib.hstu_rows8_read, lib.hstu_rows8_gemm):
    assert fn(None, None) == -1
  for fn, args in ((lib.hstu_rows8_norm, _norm_args), (lib.hstu_rows8_read, _read_args), (lib.hstu_rows8_gemm, _gemm_args)):
    assert fn(C.byref(args(rows=0)), None) == 0
  a = _gemm_args()
  a.w.rows = 0
  assert lib.hstu_rows8_gemm(C.byref(a), None) == 0


def test_library_exports_every_declared_symbol():
  text = open(os.path.join(ROOT, "include", "hstu_rows8.h")).read()
  names = sorted(set(re.findall(r"\b(?:int|const char\*) (hstu_rows8_\w+)\s*\(", text)))
  lib = _lib_rows8.load()
  assert set(names) == set(_lib_rows8.EXPORTS)
  for n in names:
    assert getattr(lib, n) is not None
  assert lib.hstu_rows8_abi_version() == _lib_rows8.ABI_VERSION


@pytest.mark.parametrize("name", ["HstuRows8", "HstuRows8NormArgs", "HstuRows8ReadArgs", "HstuRows8GemmArgs"])
def test_struct_layout_matches_header(name, tmp_path):
  struct = getattr(_lib_rows8, name)
  fields = [f[0] for f in struct._fields_]
  prog = ['#include <stdio.h>', '#include <stddef.h>', '#include "hstu_rows8.h"', "int main(void) {", f'  printf("%zu\\n", sizeof({name}));']
  prog += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["  return 0;", "}"]
  src, exe = tmp_path / "layout.c", tmp_path / "layout"
  src.write_text("\n".join(prog))
  subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
  out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
  assert int(out[0]) == C.sizeof(struct)
  for f, at in zip(fields, out[1:]):
    assert getattr(struct, f).offset == int(at), f


def test_no_cpu_path():
  x = torch.zeros((3, 128))
  codes, exponents = torch.zeros((3, 128), dtype=torch.uint8), torch.ones((1, 3, 4), dtype=torch.uint8)
  for call in (lambda: recml_amd.quantize_rows(x), lambda: recml_amd.norm_rows8(x, x[0]), lambda: recml_amd.Rows8(codes, exponents, 128)):
    with pytest.raises(ValueError, match="no CPU path"):
      call()
  with pytest.raises(TypeError, match="Rows8"):
    recml_amd.gemm_rows8(x, x)
  with pytest.raises(TypeError, match="torch.Tensor"):
    recml_amd.quantize_rows([1.0])
  with pytest.raises(ValueError, match="width"):
    recml_amd.Rows8(codes, exponents, 0)
