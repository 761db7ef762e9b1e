"""What the cache's entry points refuse, before any work (no GPU)."""

import ctypes as C

import pytest
import torch

import recml_amd
from recml_amd import _lib_serve


def _rows_args(**kw):
  a = _lib_serve.HstuKvRowsArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_serve.ABI_VERSION
  _pages(a.pages)
  a.starts, a.rows_per_seq, a.dtype, a.k, a.v = 0x1000, 3, _lib_serve.BF16, 0x2000, 0x3000
  a.k_stride_b = a.v_stride_b = 3 * 128
  a.k_stride_t = a.v_stride_t = 128
  a.k_stride_h = a.v_stride_h = 64
  return _set(a, kw)


def _attn_args(**kw):
  a = _lib_serve.HstuCachedAttnArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_serve.ABI_VERSION
  _pages(a.pages)
  a.lengths, a.rows_per_seq, a.dtype, a.q, a.out, a.max_len, a.alpha, a.inv_n = 0x1000, 1, _lib_serve.BF16, 0x2000, 0x3000, 4096, 1.0, 1.0
  a.q_stride_b = a.o_stride_b = 128
  a.q_stride_t = a.o_stride_t = 128
  a.q_stride_h = a.o_stride_h = 64
  return _set(a, kw)


def _pages(g):
  g.k_codes, g.k_scales, g.v_codes, g.v_scales, g.page_table = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
  g.n_pages, g.page_size, g.table_pages, g.B, g.H, g.d, g.bits = 128, 64, 64, 2, 2, 64, 4


def _set(a, kw):
  for name, value in kw.items():
    setattr(a.pages if hasattr(a.pages, name) else a, name, value)
  return a


PAGES = [(dict(bits=6), -4, "bits"), (dict(d=40), -4, "d=40"), (dict(d=512), -4, "d=512"), (dict(page_size=48), -4, "page_size"), (dict(page_size=0), -4, "page_size"),
         (dict(H=0), -4, "H=0"), (dict(k_codes=None), -1, "null"), (dict(v_scales=0x40008), -4, "16-byte"), (dict(page_table=None), -1, "page_table"),
         (dict(struct_size=8), -2, "struct_size"), (dict(version=99), -2, "version"), (dict(dtype=7), -4, "dtype"), (dict(rows_per_seq=-1), -4, "rows_per_seq")]


@pytest.mark.parametrize("change,status,word", PAGES + [(dict(starts=None), -1, "starts"), (dict(k=0x2004), -4, "16-byte"), (dict(v_stride_t=100), -4, "stride")])
def test_rows_refused(change, status, word):
  lib = _lib_serve.load()
  for fn in (lib.hstu_kv_write, lib.hstu_kv_read):
    assert fn(C.byref(_rows_args(**change)), None) == status
    assert word in lib.hstu_serve_last_error().decode()


@pytest.mark.parametrize("change,status,word", PAGES + [
    (dict(lengths=None), -1, "lengths"), (dict(q=0x2002), -4, "16-byte"), (dict(o_stride_h=4), -4, "stride"), (dict(max_len=0), -4, "max_len"),
    (dict(pos_tab=0x6000, pos_heads=3), -4, "pos_heads"), (dict(timestamps=0x6000), -1, "ts_tab"),
    (dict(timestamps=0x6000, ts_tab=0x7000, ts_heads=1, ts_buckets=129, ts_bucket_size=0.3), -4, "ts_buckets"),
    (dict(timestamps=0x6000, ts_tab=0x7000, ts_heads=1, ts_buckets=128, ts_bucket_size=0.0), -4, "ts_bucket_size"),
    (dict(), -5, "workspace"), (dict(workspace=0x9000, workspace_bytes=64), -5, "workspace")])
def test_attention_refused(change, status, word):
  lib = _lib_serve.load()
  assert lib.hstu_cached_attn(C.byref(_attn_args(**change)), None) == status
  assert word in lib.hstu_serve_last_error().decode()


def test_null_and_nothing_to_do():
  lib = _lib_serve.load()
  assert lib.hstu_kv_write(None, None) == -1 and lib.hstu_kv_read(None, None) == -1 and lib.hstu_cached_attn(None, None) == -1
  for change in (dict(B=0), dict(rows_per_seq=0), dict(offsets=0x9000, total_rows=0)):
    assert lib.hstu_kv_write(C.byref(_rows_args(**change)), None) == 0
    assert lib.hstu_cached_attn(C.byref(_attn_args(**change)), None) == 0
    assert lib.hstu_cached_attn_workspace_bytes(C.byref(_attn_args(**change))) == 0


def test_workspace_grows_with_what_is_split():
  lib = _lib_serve.load()
  one = lib.hstu_cached_attn_workspace_bytes(C.byref(_attn_args()))
  assert one > 0 and one % (2 * 2 * 64 * 4) == 0
  assert lib.hstu_cached_attn_workspace_bytes(C.byref(_attn_args(max_len=64))) == 0
  assert lib.hstu_cached_attn_workspace_bytes(C.byref(_attn_args(bits=3))) == 0


def test_python_refuses_cpu_tensors_and_odd_pages():
  with pytest.raises(ValueError, match="GPU"):
    recml_amd.KVPages(*(torch.zeros((2, 2, 32, 32), dtype=torch.uint8) for _ in range(4)), head_dim=64)
  with pytest.raises(ValueError, match="head_dim"):
    recml_amd.KVPages(*(torch.zeros((2, 2, 32, 32), dtype=torch.uint8) for _ in range(4)), head_dim=40)
  with pytest.raises(TypeError, match="KVPages"):
    recml_amd.kv_write(None, None, None, None, None)
  with pytest.raises(ValueError, match="bits"):
    recml_amd.KVPages.empty(1, 32, 1, 32, bits=2)


def test_header_and_binding_agree():
  import os
  import re
  header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "hstu_serve.h")).read()
  assert int(re.search(r"HSTU_SERVE_ABI_VERSION (\d+)", header).group(1)) == _lib_serve.ABI_VERSION
  assert set(re.findall(r"^(?:int|size_t|const char\*) (hstu_\w+)\(", header, re.M)) == set(_lib_serve.EXPORTS)


def _score_args(**kw):
  a = _lib_serve.HstuLogProbsArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_serve.ABI_VERSION
  a.logits, a.rows, a.stride, a.vocab, a.dtype, a.count, a.top = 0x1000, 4, 100000, 100000, _lib_serve.BF16, 1, 5
  a.tokens, a.log_probs, a.top_log_probs, a.top_tokens, a.stats, a.d_logits = 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000
  for name, value in kw.items():
    setattr(a, name, value)
  return a


@pytest.mark.parametrize("change,status,word", [
    (dict(struct_size=8), -2, "struct_size"), (dict(version=2), -2, "version"), (dict(dtype=3), -4, "dtype"), (dict(vocab=0), -4, "vocab"), (dict(rows=-1), -4, "rows"),
    (dict(top=257), -4, "top"), (dict(vocab=4), -4, "top"), (dict(logits=None), -1, "null"), (dict(tokens=None), -1, "null"), (dict(logits=0x1001), -4, "aligned"),
    (dict(rows=1 << 31), -4, "too many")])
def test_scores_refused(change, status, word):
  lib = _lib_serve.load()
  for fn in (lib.hstu_log_probs_fwd, lib.hstu_log_probs_bwd):
    assert fn(C.byref(_score_args(**change)), None) == status
    assert word in lib.hstu_serve_last_error().decode()


def test_scores_forward_and_backward_refused():
  lib = _lib_serve.load()
  for change, status in ((dict(log_probs=None), -1), (dict(top_tokens=None), -1), (dict(), -5), (dict(workspace=0x9000, workspace_bytes=16), -5)):
    assert lib.hstu_log_probs_fwd(C.byref(_score_args(**change)), None) == status
  for change, status in ((dict(stats=None), -1), (dict(d_logits=None), -1), (dict(d_logits=0x7001), -4), (dict(g_top=0x100, top_tokens=None), -1)):
    assert lib.hstu_log_probs_bwd(C.byref(_score_args(**change)), None) == status
  assert lib.hstu_log_probs_fwd(None, None) == -1 and lib.hstu_log_probs_bwd(None, None) == -1
  assert lib.hstu_log_probs_fwd(C.byref(_score_args(rows=0)), None) == 0 and lib.hstu_log_probs_workspace_bytes(C.byref(_score_args(rows=0))) == 0


def test_pages_that_32_bits_do_not_reach_are_refused():
  lib = _lib_serve.load()
  for size in ((1 << 20) + 32, 1 << 30):
    assert lib.hstu_kv_write(C.byref(_rows_args(page_size=size)), None) == -4 and "2^20" in lib.hstu_serve_last_error().decode()
    assert lib.hstu_cached_attn(C.byref(_attn_args(page_size=size)), None) == -4


def test_more_threads_than_a_launch_has_are_refused():
  """A launch counts its threads in 32 bits: 2^24 workgroups of 256, 2^26 of 64."""
  lib = _lib_serve.load()
  for fn in (lib.hstu_kv_write, lib.hstu_kv_read):
    assert fn(C.byref(_rows_args(B=1 << 20, H=16, k_stride_h=64, rows_per_seq=1)), None) == -4 and "too many" in lib.hstu_serve_last_error().decode()
  assert lib.hstu_cached_attn(C.byref(_attn_args(B=1 << 20, H=16, workspace=0x10, workspace_bytes=1 << 40)), None) == -4
  assert "too many" in lib.hstu_serve_last_error().decode()
  small = dict(vocab=16, stride=16, top=0, workspace=0x10, workspace_bytes=1 << 40)
  for change in (dict(small, rows=1 << 26), dict(small, vocab=16384, stride=16384, rows=1 << 24)):
    assert lib.hstu_log_probs_fwd(C.byref(_score_args(**change)), None) == -4 and "too many" in lib.hstu_serve_last_error().decode()


def test_more_tokens_a_row_than_the_kernels_count_are_refused():
  """2^30 of them at most: a thread's next token, and the tokens and largest entries together, are counted in 32 bits."""
  lib = _lib_serve.load()
  for count in ((1 << 30) + 1, (1 << 31) - 1):
    for fn in (lib.hstu_log_probs_fwd, lib.hstu_log_probs_bwd):
      assert fn(C.byref(_score_args(count=count, logits=None)), None) == -4 and "count" in lib.hstu_serve_last_error().decode()
    assert lib.hstu_log_probs_workspace_bytes(C.byref(_score_args(count=count))) == 0
  assert lib.hstu_log_probs_fwd(C.byref(_score_args(count=1 << 30, logits=None)), None) == -1
