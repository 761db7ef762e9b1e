"""Host side of the cache of keys and values (libhstu_serve.so): torch tensors in, HIP kernels behind the C ABI.

  KVPages            the pages of one layer: codes in 4 or 8 bits and their exponents
  kv_write           quantises new events' keys and values into the pages
  kv_read            the values that the pages stand for
  cached_attention   hstu_attention of each sequence's newest events over its kept keys and values

The attention is the layer's (recml/layers/keras/hstu.py:356-390) for the last rows of every sequence, with the keys and
values that the cache stands for.  Inference only, on a GPU only; there is no other implementation behind these names.
"""

from __future__ import annotations

import ctypes as C

import torch

from recml_amd import _lib_serve
from recml_amd import _native

HEAD_DIMS = (8, 16, 24, 32, 48, 64, 96, 128, 192, 256)
MOST_ROWS = 1 << 30          # of one sequence, and of a call's max_len: the kernels count in 32 bits
_DTYPES = {torch.bfloat16: _lib_serve.BF16, torch.float32: _lib_serve.FP32}


def _check_gpu(name, t):
  if not isinstance(t, torch.Tensor):
    raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
  if not t.is_cuda:
    raise ValueError(f"{name} must live on the GPU (got device {t.device}); this operator has no CPU path")


def _raise(lib, rc, what):
  msg = lib.hstu_serve_last_error().decode()
  if rc in (-1, -4):
    raise ValueError(f"{what} rejected the arguments ({rc}): {msg}")
  raise RuntimeError(f"{what} failed ({rc}): {msg}")


def _no_gradient(what, *tensors):
  if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _native.has_tangent(*tensors):
    raise ValueError(f"{what} has no gradient (its keys and values are codes): call it under torch.no_grad(), or train through "
                     "hstu_attention_autograd")


class KVPages:
  """The pages of one layer's cache.

  k, v: codes, uint8 [pages, heads, page_size, head_dim * bits / 8]; k_scales, v_scales: exponents, uint8
  [pages, heads, ceil(head_dim / 32), page_size].  All contiguous.  The bits (4 or 8) follow from the shapes.
  Format: include/hstu_serve.h.  Pages belong to no sequence by themselves: the calls' `page_table` [B, n] (int32) names
  the page of each sequence's places 0 .. page_size - 1, page_size .. 2 page_size - 1, ...; an entry that is no page
  (negative, say) holds nothing."""

  __slots__ = ("k", "k_scales", "v", "v_scales", "head_dim", "bits")

  def __init__(self, k, k_scales, v, v_scales, *, head_dim: int):
    d = int(head_dim)
    put = lambda bits: [object.__setattr__(self, n, t) for n, t in zip(self.__slots__, (k, k_scales, v, v_scales, d, bits))]
    for bits in (4, 8):
      if _native.check_pages(k, k_scales, v, v_scales, d, bits):
        put(bits)
        return
    if d not in HEAD_DIMS:
      raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    for name, t in (("k", k), ("k_scales", k_scales), ("v", v), ("v_scales", v_scales)):
      _check_gpu(name, t)
      if t.dtype != torch.uint8 or t.dim() != 4 or not t.is_contiguous() or t.device != k.device:
        raise ValueError(f"{name} must be a contiguous 4-d uint8 tensor on one device, got {t.dtype} {tuple(t.shape)} on {t.device}")
      if t.data_ptr() % 16:
        raise ValueError(f"{name} must start on a 16-byte boundary")
    pages, heads, size, width = k.shape
    if 8 * width not in (4 * d, 8 * d):
      raise ValueError(f"rows of {width} bytes do not hold {d} codes of 4 or 8 bits")
    if size < 32 or size % 32 or size > 1 << 20:
      raise ValueError(f"page_size must be a multiple of 32, at most 2^20, got {size}")
    if heads < 1:
      raise ValueError("there must be at least one head")
    scales = (pages, heads, (d + 31) // 32, size)
    if v.shape != k.shape or tuple(k_scales.shape) != scales or tuple(v_scales.shape) != scales:
      raise ValueError(f"k and v must share one shape and the scales be {scales}, got {tuple(k.shape)}, {tuple(v.shape)}, "
                       f"{tuple(k_scales.shape)}, {tuple(v_scales.shape)}")
    put(8 * width // d)

  def __setattr__(self, name, value):
    raise AttributeError("KVPages are what they were made of: make new ones")

  @classmethod
  def empty(cls, pages: int, page_size: int, heads: int, head_dim: int, *, bits: int = 4, device=None) -> "KVPages":
    """New pages that stand for zeros."""
    if bits not in (4, 8):
      raise ValueError(f"bits must be 4 or 8, got {bits}")
    new = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device="cuda" if device is None else device)
    codes, scales = (pages, heads, page_size, head_dim * bits // 8), (pages, heads, (head_dim + 31) // 32, page_size)
    return cls(new(*codes), new(*scales).fill_(1), new(*codes), new(*scales).fill_(1), head_dim=head_dim)

  @property
  def page_size(self) -> int:
    return self.k.shape[2]

  @property
  def heads(self) -> int:
    return self.k.shape[1]

  def _fill(self, g, page_table, B):
    g.k_codes, g.k_scales = self.k.data_ptr(), self.k_scales.data_ptr()
    g.v_codes, g.v_scales = self.v.data_ptr(), self.v_scales.data_ptr()
    g.page_table = page_table.data_ptr()
    g.n_pages, g.H, g.page_size = self.k.shape[0], self.k.shape[1], self.k.shape[2]
    g.table_pages, g.B, g.d, g.bits = page_table.shape[1], B, self.head_dim, self.bits


def _ints(name, t, device, shape=None):
  """A lengths-like tensor as the kernels read it."""
  _check_gpu(name, t)
  if t.dtype.is_floating_point or t.dtype == torch.bool or t.device != device:
    raise ValueError(f"{name} must hold integers on {device}, got {t.dtype} on {t.device}")
  if shape is not None and tuple(t.shape) != shape:
    raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
  return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _table(pages, page_table):
  if not isinstance(pages, KVPages):
    raise TypeError(f"pages must be KVPages, got {type(pages).__name__}")
  t = _ints("page_table", page_table, pages.k.device)
  if t.dim() != 2:
    raise ValueError(f"page_table must be [B, n], got {tuple(t.shape)}")
  return t


def _rows(t, unit):
  """Rows [..., H, d] with a contiguous last axis whose rows start on 16-byte boundaries (a copy when they do not)."""
  if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])):
    return t
  return t.clone(memory_format=torch.contiguous_format)


def _strides(t, jagged):
  """Batch, token and head strides; an axis of one entry has none that counts."""
  s = [st if n != 1 else 0 for st, n in zip(t.stride(), t.shape)]
  return (0, s[0], s[1]) if jagged else (s[0], s[1], s[2])


def _check_rows(name, t, pages, B, offsets, max_new):
  """Shape of new events' rows: padded [B, n, H, d], or packed [T, H, d] with `offsets` and `max_new`."""
  _check_gpu(name, t)
  if t.dtype not in _DTYPES:
    raise ValueError(f"{name}: unsupported dtype {t.dtype}: use float32 or bfloat16")
  if t.device != pages.k.device:
    raise ValueError(f"{name} is on {t.device}, the pages are on {pages.k.device}")
  tail = (pages.heads, pages.head_dim)
  if offsets is None:
    if t.dim() != 4 or t.shape[0] != B or tuple(t.shape[2:]) != tail:
      raise ValueError(f"{name} must be [{B}, n, {tail[0]}, {tail[1]}], got {tuple(t.shape)}; packed rows need `offsets` and `max_new`")
    if max_new is not None and int(max_new) != t.shape[1]:
      raise ValueError(f"max_new={max_new} does not match the {t.shape[1]} rows of a sequence")
  elif t.dim() != 3 or tuple(t.shape[1:]) != tail:
    raise ValueError(f"packed {name} must be [T, {tail[0]}, {tail[1]}], got {tuple(t.shape)}")
  elif max_new is None or not 0 <= int(max_new) <= MOST_ROWS:
    raise ValueError(f"packed rows need `max_new`, the most rows that one sequence has (up to {MOST_ROWS}), got {max_new}")


def _fill_rows(a, pages, table, B, starts, offsets, per_seq, total, k, v):
  a.struct_size, a.version = C.sizeof(_lib_serve.HstuKvRowsArgs), _lib_serve.ABI_VERSION
  pages._fill(a.pages, table, B)
  a.starts = starts.data_ptr()
  a.offsets = None if offsets is None else offsets.data_ptr()
  a.total_rows, a.rows_per_seq, a.dtype = total, per_seq, _DTYPES[k.dtype]
  a.k, a.v = k.data_ptr(), v.data_ptr()
  a.k_stride_b, a.k_stride_t, a.k_stride_h = _strides(k, offsets is not None)
  a.v_stride_b, a.v_stride_t, a.v_stride_h = _strides(v, offsets is not None)


def _call(name, a, device):
  lib = _lib_serve.load()
  with torch.cuda.device(device):
    rc = getattr(lib, name)(C.byref(a), C.c_void_p(torch.cuda.current_stream(device).cuda_stream))
  if rc != 0:
    _raise(lib, rc, name)


def kv_write(pages, k, v, page_table, starts, *, offsets=None, max_new=None) -> None:
  """Quantises the keys and values of new events into the pages.

  k, v: [B, n, H, d], or packed [T, H, d] with `offsets` [B + 1] and `max_new` (the most rows of one sequence); float32 or
  bfloat16.  Row t of sequence b goes to place starts[b] + t; rows whose place has no page are dropped.  Lengths are the
  caller's: writing the same rows again changes nothing.  Two sequences that share a page must not write it in one call."""
  if _native.kv_write(pages, k, v, page_table, starts, offsets, max_new):
    return
  table = _table(pages, page_table)
  B, device = table.shape[0], pages.k.device
  for name, t in (("k", k), ("v", v)):
    _check_rows(name, t, pages, B, offsets, max_new)
  if k.shape != v.shape or k.dtype != v.dtype:
    raise ValueError(f"k and v must share shape and dtype, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
  _no_gradient("kv_write", k, v)
  starts = _ints("starts", starts, device, (B,))
  offsets = None if offsets is None else _ints("offsets", offsets, device, (B + 1,))
  unit = 16 // k.element_size()
  k, v = _rows(k, unit), _rows(v, unit)
  a = _lib_serve.HstuKvRowsArgs()
  _fill_rows(a, pages, table, B, starts, offsets, int(max_new) if offsets is not None else k.shape[1], k.shape[0] if offsets is not None else 0, k, v)
  _call("hstu_kv_write", a, device)


def kv_read(pages, page_table, starts, *, count=None, offsets=None, max_new=None, total=None, dtype=torch.bfloat16):
  """The keys and values that the pages stand for: (k, v), [B, count, H, d] from place starts[b] on, or packed
  [total, H, d] with `offsets` [B + 1] and `max_new` (rows of no sequence are not written).  Exact in float32, and in bfloat16
  down to its smallest values.  Places without a page read as zeros."""
  if dtype is torch.bfloat16 or dtype is torch.float32:
    got = _native.kv_read(pages, page_table, starts, count, offsets, max_new, total, dtype is torch.float32)
    if got is not None:
      return got
  table = _table(pages, page_table)
  B, device = table.shape[0], pages.k.device
  if dtype not in _DTYPES:
    raise ValueError(f"unsupported dtype {dtype}: use float32 or bfloat16")
  starts = _ints("starts", starts, device, (B,))
  if offsets is None:
    if count is None or not 0 <= int(count) <= MOST_ROWS or total is not None or max_new is not None:
      raise ValueError("pass `count`, or `offsets` with `max_new` and `total`")
    shape, per_seq = (B, int(count)), int(count)
  else:
    if count is not None or max_new is None or total is None or not 0 <= int(max_new) <= MOST_ROWS or int(total) < 0:
      raise ValueError("pass `count`, or `offsets` with `max_new` and `total`")
    offsets = _ints("offsets", offsets, device, (B + 1,))
    shape, per_seq = (int(total),), int(max_new)
  k, v = (torch.empty((*shape, pages.heads, pages.head_dim), dtype=dtype, device=device) for _ in range(2))
  a = _lib_serve.HstuKvRowsArgs()
  _fill_rows(a, pages, table, B, starts, offsets, per_seq, shape[0] if offsets is not None else 0, k, v)
  _call("hstu_kv_read", a, device)
  return k, v


def _bias_table(name, t, heads, width, device):
  _check_gpu(name, t)
  if t.dim() == 1:
    t = t.unsqueeze(0)
  if t.dim() != 2 or t.shape[0] not in (1, heads) or t.device != device:
    raise ValueError(f"{name} must be [n] or [1|{heads}, n] on {device}, got {tuple(t.shape)} on {t.device}")
  if width is not None and t.shape[1] != width:
    raise ValueError(f"{name} must have {width} entries per head, got {t.shape[1]}")
  return t.to(torch.float32).contiguous()


def cached_attention(q, pages, page_table, lengths, *, max_len, offsets=None, max_new=None, n=None, alpha=1.0, pos_bias=None,
                     timestamps=None, ts_bias=None, ts_bucket_size=0.301, out=None):
  """The rows that hstu_attention (causal) has for each sequence's newest events, over the keys and values in `pages`.

  Args:
    q: the newest events' queries, [B, m, H, d], or packed [T, H, d] with `offsets` [B + 1] and `max_new` (the most rows of
      one sequence); float32 or bfloat16.  With m rows of a sequence of lengths[b] events, row t is the event at place
      i = lengths[b] - m + t and attends to the places j <= i; rows at places below 0 are zeros.
    pages, page_table: the cache, with the new events written (kv_write).
    lengths: int [B], how many events each sequence has, the new ones included.
    max_len: the length L of the full call that this stands for: the default normaliser and the tables' extent.  Places at or
      past it, or past the page table's end, are not there; rows at them are zeros.
    n: the normaliser (default max_len); alpha: the logit scale.
    pos_bias: [2L - 1] or [H, 2L - 1]; logit (i, j) gets pos_bias[(L - 1) + j - i].
    timestamps, ts_bias: int64 [B, L] and [nb + 1] or [H, nb + 1] (at most 128 buckets); logit (i, j) gets
      ts_bias[bucket(ts[min(i + 1, lengths[b] - 1)] - ts[j])].
    out: optional preallocated output.  Packed rows of no sequence are left as they were in it.

  Returns: a tensor shaped and typed like q.  Inference only: raises where a gradient is asked for."""
  got = _native.cached_attention(q, pages, page_table, lengths, max_len, offsets, max_new, n, alpha, pos_bias, timestamps, ts_bias, ts_bucket_size, out)
  if got is not None:
    return got
  table = _table(pages, page_table)
  B, device, H = table.shape[0], pages.k.device, pages.heads
  _check_rows("q", q, pages, B, offsets, max_new)
  _no_gradient("cached_attention", q, pos_bias, ts_bias, out)
  lengths = _ints("lengths", lengths, device, (B,))
  offsets = None if offsets is None else _ints("offsets", offsets, device, (B + 1,))
  L = int(max_len)
  if not 1 <= L <= MOST_ROWS:
    raise ValueError(f"max_len must lie between 1 and {MOST_ROWS}, got {max_len}")
  n = L if n is None else n
  if not n > 0:
    raise ValueError(f"normaliser n must be positive, got {n}")
  unit = 16 // q.element_size()
  q = _rows(q, unit)
  if out is None:
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
  else:
    _check_gpu("out", out)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != device:
      raise ValueError(f"out must be a {q.dtype} tensor of shape {tuple(q.shape)} on {device}")
    if _rows(out, unit) is not out or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
      raise ValueError("out's rows must be contiguous, start on 16-byte boundaries and lie apart")
  a = _lib_serve.HstuCachedAttnArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_serve.ABI_VERSION
  pages._fill(a.pages, table, B)
  a.lengths, a.offsets = lengths.data_ptr(), None if offsets is None else offsets.data_ptr()
  a.total_rows, a.rows_per_seq, a.dtype = (q.shape[0], int(max_new), _DTYPES[q.dtype]) if offsets is not None else (0, q.shape[1], _DTYPES[q.dtype])
  a.q, a.out = q.data_ptr(), out.data_ptr()
  a.q_stride_b, a.q_stride_t, a.q_stride_h = _strides(q, offsets is not None)
  a.o_stride_b, a.o_stride_t, a.o_stride_h = _strides(out, offsets is not None)
  a.max_len, a.alpha, a.inv_n = L, float(alpha), 1.0 / float(n)
  keep = []
  if pos_bias is not None:
    pt = _bias_table("pos_bias", pos_bias, H, 2 * L - 1, device)
    keep.append(pt)
    a.pos_tab, a.pos_heads = pt.data_ptr(), pt.shape[0]
  if (timestamps is None) != (ts_bias is None):
    raise ValueError("Both or neither of `timestamps` and `ts_bias` must be provided.")
  if ts_bias is not None:
    tt = _bias_table("ts_bias", ts_bias, H, None, device)
    _check_gpu("timestamps", timestamps)
    if tuple(timestamps.shape) != (B, L) or timestamps.device != device:
      raise ValueError(f"timestamps must be [{B}, {L}] on {device}, got {tuple(timestamps.shape)} on {timestamps.device}")
    if not 1 <= tt.shape[1] <= 129:
      raise ValueError(f"ts_bias may have up to 129 entries per head (128 buckets), got {tt.shape[1]}")
    ts = timestamps.to(torch.int64).contiguous()
    keep += [tt, ts]
    a.timestamps, a.ts_tab = ts.data_ptr(), tt.data_ptr()
    a.ts_heads, a.ts_buckets, a.ts_bucket_size = tt.shape[0], tt.shape[1] - 1, float(ts_bucket_size)
  need = _lib_serve.load().hstu_cached_attn_workspace_bytes(C.byref(a))
  if need:
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    keep.append(ws)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
  _call("hstu_cached_attn", a, device)
  del keep
  return out
