"""A block's steps on rows kept in 8 bits (libhstu_rows8.so): torch tensors in, HIP kernels behind the C ABI.

  Rows8            rows of activations, or a weight's output columns, as e4m3 codes with a power of two for each block of 128
  quantize_rows    rows as they are into 8 bits
  norm_rows8       layer norm or root-mean-square norm into 8 bits, with the residual's addition and the U gate
                   (recml/layers/keras/hstu.py:442, 471-472)
  gemm_rows8       the product of two of them, with bias, residual and SiLU (recml/layers/keras/hstu.py:444-449, 473-474)

What layer_norm, norm_gate and gemm_silu do in bf16, for inference with half the bytes and twice the matrix cores' rate.  On a GPU only;
there is no other implementation behind these names.
"""

from __future__ import annotations

import ctypes as C

import torch

from recml_amd import _lib_rows8
from recml_amd import _native

BLOCK = 128
MAX_WIDTH = _lib_rows8.MAX_WIDTH
MAX_ROWS = (1 << 31) - 1
_DTYPES = {torch.bfloat16: _lib_rows8.BF16, torch.float32: _lib_rows8.FP32}


def _check_gpu(name, t):
  if not isinstance(t, torch.Tensor):
    raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
  if not t.is_cuda:
    raise ValueError(f"{name} must live on the GPU (got device {t.device}); this operator has no CPU path")


def _check_like(name, t, shape, dtype, device):
  _check_gpu(name, t)
  if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device:
    raise ValueError(f"{name} must be {dtype} {tuple(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _no_gradient(what, *tensors):
  if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _native.has_tangent(*tensors):
    raise ValueError(f"{what} has no gradient (its rows are codes): call it under torch.no_grad(), or train through layer_norm, norm_gate and "
                     "gemm_silu")


def _call(name, args, device):
  lib = _lib_rows8.load()
  with torch.cuda.device(device):
    rc = getattr(lib, name)(C.byref(args), C.c_void_p(torch.cuda.current_stream(device).cuda_stream))
  if rc != 0:
    msg = lib.hstu_rows8_last_error().decode()
    if rc in (-1, -4):
      raise ValueError(f"{name} rejected the arguments ({rc}): {msg}")
    raise RuntimeError(f"{name} failed ({rc}): {msg}")


def _new(kind):
  a = kind()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  return a


def _shapes(rows, width):
  blocks = -(-width // BLOCK)
  return (rows, BLOCK * blocks), (-(-blocks // 4), rows, 4)


class Rows8:
  """Rows in 8 bits.

  codes: uint8 [rows, 128 ceil(width / 128)], e4m3, zeros past the width; exponents: uint8 [ceil(width / 512), rows, 4], the biased powers of
  two (1 to 246) of four blocks of 128 side by side (255: the block stands for NaN).  Both contiguous, on one device.  Format:
  include/hstu_rows8.h.  A weight [K, N] is kept as its N output columns: quantize_rows(w.t())."""

  __slots__ = ("codes", "exponents", "width")

  def __init__(self, codes, exponents, width: int):
    if not _native.check_rows8(codes, exponents, width):
      width = int(width)
      if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"width must lie between 1 and {MAX_WIDTH}, got {width}")
      for name, t, dims in (("codes", codes, 2), ("exponents", exponents, 3)):
        _check_gpu(name, t)
        if t.dtype != torch.uint8 or t.dim() != dims or not t.is_contiguous() or t.device != codes.device:
          raise ValueError(f"{name} must be a contiguous {dims}-d uint8 tensor on one device, got {t.dtype} {tuple(t.shape)} on {t.device}")
      want = _shapes(codes.shape[0], width)
      if (tuple(codes.shape), tuple(exponents.shape)) != want or codes.shape[0] > MAX_ROWS:
        raise ValueError(f"rows of {width} values are codes {want[0]} and exponents {want[1]}, got {tuple(codes.shape)} and {tuple(exponents.shape)}")
      if codes.data_ptr() % 16 or exponents.data_ptr() % 4:
        raise ValueError("codes must start on a 16-byte boundary and exponents on a 4-byte one")
    self._put(codes, exponents, width)

  def _put(self, codes, exponents, width):
    _set_codes(self, codes)
    _set_exponents(self, exponents)
    _set_width(self, width)
    return self

  def __setattr__(self, name, value):
    raise AttributeError("Rows8 are what they were made of: make new ones")

  def __reduce__(self):
    return _loaded, (self.codes, self.exponents, self.width)

  def __repr__(self):
    return f"Rows8({self.rows} rows of {self.width} on {self.codes.device})"

  @classmethod
  def _of(cls, codes, exponents, width):
    return object.__new__(cls)._put(codes, exponents, width)

  @classmethod
  def _empty(cls, rows, width, device):
    if not 1 <= width <= MAX_WIDTH:
      raise ValueError(f"rows must have 1 to {MAX_WIDTH} values, got {width}")
    if rows > MAX_ROWS:
      raise ValueError(f"at most {MAX_ROWS} rows, got {rows}")
    return cls._of(*(torch.empty(s, dtype=torch.uint8, device=device) for s in _shapes(rows, width)), width)

  @property
  def rows(self) -> int:
    return self.codes.shape[0]

  @property
  def device(self):
    return self.codes.device

  def values(self, dtype=torch.bfloat16):
    """What the rows stand for, [rows, width]: exact in float32, and in bfloat16 down to its smallest values."""
    got = _native.read_rows8(self.codes, self.exponents, self.width, dtype)
    if got is not None:
      return got
    _check_gpu("codes", self.codes)
    if dtype not in _DTYPES:
      raise ValueError(f"dtype must be torch.bfloat16 or torch.float32, got {dtype}")
    out = torch.empty((self.rows, self.width), dtype=dtype, device=self.device)
    a = _new(_lib_rows8.HstuRows8ReadArgs)
    self._fill(a.rows)
    a.out, a.out_stride, a.dtype = out.data_ptr(), self.width, _DTYPES[dtype]
    _call("hstu_rows8_read", a, self.device)
    return out

  def _fill(self, r):
    r.codes, r.exponents, r.rows, r.width = self.codes.data_ptr(), self.exponents.data_ptr(), self.rows, self.width


def _loaded(codes, exponents, width):
  """Rows8 that were copied or saved.  On a GPU they are checked as new ones are; elsewhere (a file loaded with map_location="cpu") they are kept,
  and refused where something is asked of them."""
  return Rows8(codes, exponents, width) if codes.is_cuda else Rows8._of(codes, exponents, width)


_set_codes, _set_exponents, _set_width = (getattr(Rows8, name).__set__ for name in Rows8.__slots__)      # (past __setattr__)


def _flat(t):
  """[..., W] as [rows, W] with one row stride (a copy when the layout does not allow it)."""
  W = t.shape[-1]
  if t.stride(-1) != 1 and W > 1:
    t = t.contiguous()
  return t if t.dim() == 2 else t.reshape(-1, W)


def _norm(what, x, gamma, beta, eps, gate, add, kind):
  got = _native.norm_rows8(x, gamma, beta, eps, gate, add, kind)
  if got is not None:
    return Rows8._of(*got[:3]), got[3]
  _check_gpu("x", x)
  if x.dtype not in _DTYPES:
    raise ValueError(f"x: unsupported dtype {x.dtype}: use float32 or bfloat16")
  if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
    raise ValueError(f"x must be [..., W] with W from 1 to {MAX_WIDTH}, got {tuple(x.shape)}")
  W, dev = x.shape[-1], x.device
  for name, t in (("gate", gate), ("add", add)):
    if t is not None:
      _check_like(name, t, x.shape, x.dtype, dev)
  keep = {}
  for name, t in (("gamma", gamma), ("beta", beta)):
    if t is not None:
      _check_gpu(name, t)
      _check_like(name, t.reshape(-1), (W,), x.dtype, dev)
      keep[name] = t.reshape(-1).contiguous()
  if kind != _lib_rows8.AS_IS and gamma is None:
    raise ValueError("a norm needs gamma")
  _no_gradient(what, x, gamma, beta, gate, add)
  for name, t in (("x", x), ("gate", gate), ("add", add)):
    if t is not None:
      keep[name] = _flat(t)
  R = keep["x"].shape[0]
  rows = Rows8._empty(R, W, dev)
  total = None if add is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
  a = _new(_lib_rows8.HstuRows8NormArgs)
  rows._fill(a.rows)
  a.norm, a.dtype, a.eps = kind, _DTYPES[x.dtype], float(eps)
  for name, t in keep.items():
    setattr(a, name, t.data_ptr())
    if t.dim() == 2:
      setattr(a, name + "_stride", t.stride(0) if R > 1 else 0)
  if total is not None:
    a.sum, a.sum_stride = total.data_ptr(), W
  _call("hstu_rows8_norm", a, dev)
  return rows, total


def quantize_rows(x) -> Rows8:
  """Rows in 8 bits: x [..., W], float32 or bfloat16 (a copy is made where the last axis is not contiguous or the others do not flatten to
  one row stride), as they are.  The leading axes become one.  A weight [K, N] is quantised as quantize_rows(w.t()).

  Every value is off by at most 2^-4 of itself, or half the smallest step of its block of 128 (2^-17 of the block's largest value at most); a
  block that holds a value which is not finite stands for NaN."""
  return _norm("quantize_rows", x, None, None, 0.0, None, None, _lib_rows8.AS_IS)[0]


def renew(kept, fresh):
  """`fresh` (Rows8, a tensor or None) in the place of `kept`, so that what reads it there (a captured graph) reads the new one; or as it is, where
  that is of another kind or size, or elsewhere."""
  if isinstance(fresh, Rows8):
    if not isinstance(kept, Rows8) or (kept.rows, kept.width, kept.device) != (fresh.rows, fresh.width, fresh.device):
      return fresh
    renew(kept.codes, fresh.codes)
    renew(kept.exponents, fresh.exponents)
    return kept
  if fresh is None or kept is None or (kept.shape, kept.dtype, kept.device) != (fresh.shape, fresh.dtype, fresh.device):
    return fresh
  with torch.inference_mode():                     # (`kept` may have been made there)
    return kept.copy_(fresh)


def norm_rows8(x, gamma, beta=None, eps: float = 1e-6, *, gate=None, add=None, rms: bool = False):
  """A norm of rows over their last axis, in 8 bits: gate * layer_norm(x + add), statistics and products in fp32, or in 64 bits for float32 rows, one
  rounding.  (A row whose sum of squares, for float32 their mean, is past fp32's largest comes back as zeros, times gamma, plus beta.)

  Args:
    x: [..., W], float32 or bfloat16 (a copy is made where the last axis is not contiguous or the others do not flatten to one row
      stride; a slice of a fused projection does).  The leading axes become one.
    gamma, beta: W values of x's type; beta may be None.
    gate: shaped like x: multiplied with the normed rows (the block's U).
    add: shaped like x: added before the norm (a residual).  The sum, rounded to x's type, is what is normed, and is returned too.
    rms: the root-mean-square norm, without the mean: x / sqrt(mean(x^2) + eps) * gamma (+ beta).

  Returns Rows8, or with `add` (Rows8, x + add).  Inference only."""
  rows, total = _norm("norm_rows8", x, gamma, beta, eps, gate, add, _lib_rows8.RMS if rms else _lib_rows8.LAYER)
  return rows if add is None else (rows, total)


def gemm_rows8(x, w, bias=None, activation: bool = False, *, residual=None, dtype=torch.bfloat16):
  """act(x @ w.T + residual + bias): x Rows8 [M, K], w Rows8 [N, K] (a weight's output columns) -> [M, N] of `dtype` (bfloat16 or
  float32), sums in fp32, one rounding.  bias [N], residual [M, N] (row stride free) of `dtype`; activation: silu, last.  With float32
  results every product of what the rows stand for is exact (of values to the nearest multiple of 2^-133 in blocks under 2^-116); with bfloat16 ones each is cut to 2^-13 of the largest of its eight neighbours along
  K, as the matrix instructions on codes do (2e-5 of a result in the mean square beside the 1.7e-3 of its
  rounding: 1.5 % of results are the exact value's other neighbour).  Inference only."""
  if isinstance(x, Rows8) and isinstance(w, Rows8) and x.width == w.width:
    got = _native.gemm_rows8(x.codes, x.exponents, w.codes, w.exponents, x.width, bias, activation, residual, dtype)
    if got is not None:
      return got
  for name, t in (("x", x), ("w", w)):
    if not isinstance(t, Rows8):
      raise TypeError(f"{name} must be Rows8, got {type(t).__name__}")
    _check_gpu(f"{name}.codes", t.codes)
  if x.width != w.width or x.device != w.device:
    raise ValueError(f"x [M, K] and w [N, K] on one device expected, got rows of {x.width} on {x.device} and of {w.width} on {w.device}")
  if dtype not in _DTYPES:
    raise ValueError(f"dtype must be torch.bfloat16 or torch.float32, got {dtype}")
  M, N, dev = x.rows, w.rows, x.device
  if bias is not None:
    _check_gpu("bias", bias)
    bias = bias.reshape(-1)
    _check_like("bias", bias, (N,), dtype, dev)
    bias = bias.contiguous()
  if residual is not None:
    _check_like("residual", residual, (M, N), dtype, dev)
  _no_gradient("gemm_rows8", bias, residual)
  out = torch.empty((M, N), dtype=dtype, device=dev)
  a = _new(_lib_rows8.HstuRows8GemmArgs)
  x._fill(a.x)
  w._fill(a.w)
  a.dtype, a.activation, a.out, a.out_stride = _DTYPES[dtype], 1 if activation else 0, out.data_ptr(), N
  if bias is not None:
    a.bias = bias.data_ptr()
  if residual is not None:
    residual = _flat(residual)
    a.c, a.c_stride = residual.data_ptr(), residual.stride(0) if M > 1 else 0
  _call("hstu_rows8_gemm", a, dev)
  return out
