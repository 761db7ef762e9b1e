"""Log probabilities of many short rows, where a wave takes a row, and around the borders of that, against 64 bits."""

import math

import pytest
import torch

import recml_amd
from tests import serve_reference as R
from tests.test_gpu_log_probs import BF16, F32, STEP, _check, _gen, _logits, _sums_off

pytestmark = pytest.mark.gpu

# (a wave holds 512 vectors: 4096 entries in bf16, 2048 in fp32, less where rows start between two vectors; its list 256 entries)
WIDTHS = [(BF16, v) for v in (1, 63, 256, 257, 300, 399, 701, 2047, 4088, 4089, 4096, 4097)] + [(F32, v) for v in (1, 63, 257, 300, 701, 2044, 2045, 2048, 2049)]


@pytest.mark.parametrize("top", [0, 17, 50, 51])
@pytest.mark.parametrize("dtype,vocab", WIDTHS)
def test_forward_of_many_rows(gpu, dtype, vocab, top):
  rows = 1024 if vocab > 1000 else 1100
  x = _logits(rows, vocab, dtype, vocab)
  x[5, vocab // 2 :] = -math.inf
  x[7, vocab // 3] = math.nan
  tokens = torch.randint(-1, vocab + 1, (rows, 3), generator=_gen(1))
  tokens[7] = tokens[7].clamp(min=0)
  top = min(top, vocab)
  _check(recml_amd.token_log_probs(x.cuda(), tokens.cuda(), top=top, entropy=True), x, tokens, top, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1023, 1024, 4095, 4096])
def test_rows_of_fewer_vectors_than_entries_asked_for(gpu, rows, dtype):
  """No bound holds the list: every entry is ranked or found bit by bit, on one wave and on four."""
  for vocab in (256, 264, 300, 392):
    x = _logits(rows, vocab, dtype, vocab + rows)
    x[3] = x[3, 0]
    _check(recml_amd.token_log_probs(x.cuda(), top=50), x, None, 50, False)


@pytest.mark.parametrize("dtype,vocab,count,top", [
    (BF16, 63, 2, 0), (BF16, 300, 5, 50), (BF16, 701, 70, 17), (BF16, 2047, 200, 10), (BF16, 4089, 3, 50), (BF16, 4097, 2, 51),
    (F32, 63, 2, 5), (F32, 300, 5, 50), (F32, 701, 70, 17), (F32, 2045, 200, 50), (F32, 2049, 2, 51)])
def test_gradients_of_many_rows(gpu, dtype, vocab, count, top):
  rows = 1024
  x = _logits(rows, vocab, dtype, vocab + 1)
  x[9, vocab // 2 :] = -math.inf
  tokens = torch.randint(-1, vocab, (rows, count), generator=_gen(2))
  tokens[:, -1] = tokens[:, 0]                      # the same token twice
  tokens[2] = -1                                    # a row that asks for nothing
  tokens[9] = tokens[9].clamp(max=vocab // 2 - 1)
  g = [torch.randn(s, generator=_gen(3 + i)) for i, s in enumerate([(rows, count), (rows,), (rows, top)])]
  if top > vocab // 2:
    g[2][9] = 0.0
  xs = x.cuda().requires_grad_(True)
  got = recml_amd.token_log_probs(xs, tokens.cuda(), top=top, entropy=True)
  outs = [(got.log_probs, g[0]), (got.entropy, g[1])] + ([(got.top_log_probs, g[2])] if top else [])
  d = torch.autograd.grad([o for o, _ in outs], xs, [t.cuda() for _, t in outs])[0].cpu()
  want = R.log_probs(x, tokens, top, *(g if top else g[:2]))
  lp, inner = want[5], want[6]
  p = lp.exp()
  # an entry's own gradients: as many roundings of partial sums up to their size as it has (at most all of the row's); p is off by its
  # exponent's error, the sum of gradients by its additions, the entropy's part by the entropy's error
  size = sum(t.double().abs().reshape(rows, -1).sum(-1, keepdim=True) for t in g)
  off = 8 * STEP * lp.abs().nan_to_num(posinf=0) + 3 * _sums_off(vocab)
  tol = p * (inner.abs() * off + size * (8 * _sums_off(vocab) * (1 + math.log(vocab + 1)))) + 4 * STEP * (size * p + want[4].abs()) + 2.0**-132
  tol = tol + torch.finfo(dtype).eps / 2 * want[4].abs() + STEP * (count + top) * size * p
  mine = torch.zeros((rows, vocab), dtype=torch.float64)
  times = torch.zeros((rows, vocab), dtype=torch.float64)
  for ids, own in ((tokens, g[0]), (want[3], g[2])):
    there = (ids >= 0).double()
    mine.scatter_add_(1, ids.clamp(min=0), own.double().abs() * there)
    times.scatter_add_(1, ids.clamp(min=0), there)
  tol = tol + STEP * times * mine
  bad = (d.double() - want[4]).abs() > tol
  assert not bad.any(), (float((d.double() - want[4]).abs().max()), int(bad.sum()))
  assert not d[9, vocab // 2 :].any()


def test_a_refused_call_raises_the_same_either_way(gpu):
  """More threads than a launch counts, through the native call and through Python's; and a bucket size that is nothing in fp32."""
  x = torch.zeros((1, 1)).cuda().expand(1 << 26, 1)
  for entropy in (True, 1):                          # (1: not the native call's)
    with pytest.raises(ValueError, match="too many"):
      recml_amd.token_log_probs(x, entropy=entropy)
  pages = recml_amd.KVPages.empty(1, 32, 1, 8)
  table, q = torch.zeros((1, 1), dtype=torch.int32).cuda(), torch.zeros((1, 1, 1, 8)).cuda()
  for lengths in (torch.ones(1, dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.int64).cuda()):     # (the second is Python's)
    with pytest.raises(ValueError, match="ts_bucket_size"):
      recml_amd.cached_attention(q, pages, table, lengths, max_len=4, timestamps=torch.zeros((1, 4), dtype=torch.int64).cuda(), ts_bias=torch.zeros(9).cuda(),
                                 ts_bucket_size=1e-60)


def test_inside_inference_mode(gpu):
  """Tensors that keep no version: the same results."""
  x = _logits(3, 500, BF16, 1).cuda()
  want = recml_amd.token_log_probs(x, torch.tensor([1, 2, 3]).cuda(), top=4, entropy=True)
  with torch.inference_mode():
    y = x.clone()
    got = recml_amd.token_log_probs(y, torch.tensor([1, 2, 3]).cuda(), top=4, entropy=True)
    model = recml_amd.HSTU(vocab_size=50, max_positions=32, model_dim=16, num_heads=2, num_layers=2, device="cuda:0", seed=3).eval()
    ids, ts = torch.randint(0, 50, (2, 8), generator=_gen(2)).cuda(), torch.arange(16).reshape(2, 8).cuda() * 1000
    tab = torch.randn((129,), generator=_gen(3)).cuda()
    cache = model.new_cache(2, 32, timestamps=True)
    model.prefill(ids[:, :4], cache, seq_lens=torch.tensor([4, 2]).cuda(), timestamps=ts[:, :4], ts_bias=tab)
    out = model.extend(ids[:, 4:], cache, timestamps=ts[:, 4:], ts_bias=tab)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  cache = model.new_cache(2, 32, timestamps=True)
  model.prefill(ids[:, :4], cache, seq_lens=torch.tensor([4, 2]).cuda(), timestamps=ts[:, :4], ts_bias=tab)
  assert torch.equal(out, model.extend(ids[:, 4:], cache, timestamps=ts[:, 4:], ts_bias=tab))
