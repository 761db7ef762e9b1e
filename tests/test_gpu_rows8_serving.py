"""A quantised model's prefill, extend and packed forward are the runs of the operators on its weights in 8 bits, head included, bit by bit."""

import pytest
import torch

import recml_amd
from tests.test_gpu_rows8_model import _by_hand, _gen, _model

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _norm(model, x):
  if x.dtype == BF16:
    return recml_amd.layer_norm(x, model.final_norm_gamma, model.final_norm_beta, model.eps)
  return torch.nn.functional.layer_norm(x, (model.model_dim,), model.final_norm_gamma, model.final_norm_beta, model.eps)


def _front(model, ids, places):
  """Rows [T, D] of ids [T] at their places."""
  scale = model.model_dim**0.5
  if model.item_embedding.dtype == BF16:
    return recml_amd.embed_norm(ids, model.item_embedding, model.final_norm_gamma, model.final_norm_beta, model.eps, scale=scale, positions=places,
                                pos_table=model.position_embedding)
  return _norm(model, model.item_embedding[ids] * scale + model.position_embedding[places])


def _head(model, x):
  x = _norm(model, x)
  if model.reverse_embedding is None:
    return x
  return recml_amd.gemm_rows8(recml_amd.quantize_rows(x), recml_amd.quantize_rows(model.reverse_embedding.t()), dtype=x.dtype)


def _whole(model, ids, lens, cache, max_len):
  """Packed rows of whole histories, written to `cache` if there is one; the outputs [T, ...]."""
  B, L = ids.shape
  rows = torch.cat([ids[b, : int(n)] for b, n in enumerate(lens.tolist())])
  places = torch.cat([torch.arange(int(n), device=ids.device) for n in lens.tolist()])
  offsets = torch.zeros(B + 1, dtype=torch.int32, device=ids.device)
  offsets[1:] = torch.cumsum(lens, 0)
  x = _front(model, rows, places)
  for i, block in enumerate(model.decoder_blocks):
    def attend(q, k, v):
      if cache is not None:
        recml_amd.kv_write(cache.layers[i], k, v, cache.page_table, torch.zeros(B, dtype=torch.int32, device=ids.device), offsets=offsets, max_new=L)
      return recml_amd.hstu_attention(q, k, v, seq_offsets=offsets, max_len=max_len, n=float(max_len))
    x = _by_hand(block, x, attend)
  return _head(model, x)


@pytest.mark.parametrize("head", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_forward(gpu, dtype, head):
  model = _model(dtype, head=head)
  model.quantize(head=head)
  ids, lens = torch.randint(0, 300, (4, 33), generator=_gen(3)).to(gpu), torch.tensor([33, 0, 5, 20], dtype=torch.int32, device=gpu)
  got, want = model(ids, seq_lens=lens, jagged=True), _whole(model, ids, lens, None, 33)
  assert torch.equal(torch.cat([got[b, : int(n)] for b, n in enumerate(lens.tolist())]), want)


@pytest.mark.parametrize("head", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_prefill_and_extend(gpu, bits, dtype, head):
  model = _model(dtype, head=head, use_bias=True)
  model.quantize(head=head)
  B, L, H, hd = 3, 40, 2, 32
  ids, lens = torch.randint(0, 300, (B, 25), generator=_gen(3)).to(gpu), torch.tensor([25, 1, 17], dtype=torch.int32, device=gpu)
  cache, other = (model.new_cache(B, L, bits=bits, page_size=32) for _ in range(2))
  got, want = model.prefill(ids, cache, seq_lens=lens), _whole(model, ids, lens, other, L)
  assert torch.equal(torch.cat([got[b, : int(n)] for b, n in enumerate(lens.tolist())]), want)
  starts = lens.clone()
  for n in (1, 2, 1):
    new = torch.randint(0, 300, (B, n), generator=_gen(10 + int(starts[0]))).to(gpu)
    got = model.extend(new, cache)
    x = _front(model, new.reshape(-1), (starts[:, None] + torch.arange(n, device=gpu)).reshape(-1).long())
    for i, block in enumerate(model.decoder_blocks):
      def attend(q, k, v):
        to4 = lambda t: t.reshape(B, n, H, hd)
        recml_amd.kv_write(other.layers[i], to4(k), to4(v), other.page_table, starts)
        return recml_amd.cached_attention(to4(q), other.layers[i], other.page_table, starts + n, max_len=L)
      x = _by_hand(block, x, attend)
    assert torch.equal(got.reshape(B * n, -1), _head(model, x))
    starts = starts + n
  assert torch.equal(cache.lengths.to(starts), starts)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_of_a_quantised_head(gpu, dtype):
  model = _model(dtype)
  model.quantize(head=True)
  ids, lens = torch.randint(0, 300, (4, 33), generator=_gen(3)).to(gpu), torch.tensor([33, 1, 5, 20], dtype=torch.int32, device=gpu)
  want = recml_amd.token_log_probs(model(ids, seq_lens=lens), ids)
  got = model.log_probs(ids, ids, seq_lens=lens)
  assert torch.equal(got.log_probs, want.log_probs)
