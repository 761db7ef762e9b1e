"""Loads the native host sides (recml_amd/lib/_native.so, built from recml_amd/csrc/native.cpp, and, for the serving operators,
_native_serve.so from native_serve.cpp).

Its functions take a call whose arguments are ready for the kernels as they are, and return None for any other, which
the Python side then checks, converts or reports.
"""

from __future__ import annotations

import importlib.util
import os

import torch
from torch.autograd import forward_ad

from recml_amd import _lib, _lib_block, _lib_serve

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_native.so")


def has_tangent(*tensors) -> bool:
  """Whether one of the tensors carries a forward-mode tangent: the kernels' results have none, so such a call goes through the
  autograd functions, which refuse it."""
  return any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _load(name, *libraries):
  path = os.path.join(os.path.dirname(PATH), name + ".so")
  if not os.path.exists(path):
    raise RuntimeError(f"{path} is missing: build it with `python -m recml_amd.build`; this package has no CPU fallback")
  for library in libraries:
    library.load()
  spec = importlib.util.spec_from_file_location("recml_amd.lib." + name, path)
  module = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(module)
  return module


def _other_library() -> bool:
  """Whether other libraries than the packaged ones are to run: every call then goes the Python way."""
  return bool(os.environ.get("RECML_AMD_LIB") or os.environ.get("RECML_AMD_BLOCK_LIB"))


def _other_serve_library() -> bool:
  return bool(os.environ.get("RECML_AMD_SERVE_LIB"))


def _decline(*args):
  return None


def _first_call(name, functions, load, other):
  """A stand-in that loads the module when it is first called and is replaced by the module's function."""

  def call(*args):
    module = None if other() else load()
    for n in functions:
      globals()[n] = _decline if module is None else getattr(module, n)
    return globals()[name](*args)

  return call


_FUNCTIONS = ("attention", "block", "blocks", "embed", "final_norm", "linear", "pack", "mask_lengths", "raised", "norm_gate_bwd", "has_room")
attention, block, blocks, embed, final_norm, linear, pack, mask_lengths, raised, norm_gate_bwd, has_room = (
    _first_call(n, _FUNCTIONS, lambda: _load("_native", _lib, _lib_block), _other_library) for n in _FUNCTIONS)

_SERVE_FUNCTIONS = ("check_pages", "kv_write", "kv_read", "cached_attention", "token_log_probs", "accumulators")
check_pages, kv_write, kv_read, cached_attention, token_log_probs, accumulators = (
    _first_call(n, _SERVE_FUNCTIONS, lambda: _load("_native_serve", _lib_serve), _other_serve_library) for n in _SERVE_FUNCTIONS)
