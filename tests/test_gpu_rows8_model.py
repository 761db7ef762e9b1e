"""HSTU's blocks with their weights in 8 bits: every form of their calls is the run of the operators, and what is refused."""

import copy
import io

import pytest
import torch

import recml_amd

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _model(dtype, D=64, H=2, layers=2, vocab=300, positions=64, head=True, seed=3, use_bias=False):
  m = recml_amd.HSTU(vocab_size=vocab, max_positions=positions, model_dim=D, num_heads=H, num_layers=layers, add_head=head, dtype=dtype, device="cuda:0", seed=seed,
                     scale_by_sqrt_dim=True)
  if use_bias:
    m.decoder_blocks = torch.nn.ModuleList(recml_amd.HSTUBlock(D, H, use_bias=True, dtype=dtype, device="cuda:0", generator=_gen(seed + i)) for i in range(layers))
  g = _gen(seed + 1)
  with torch.no_grad():
    for p in m.parameters():
      p.add_((torch.randn(p.shape, generator=g) * 0.05).to(p))
  return m.eval()


def _by_hand(block, rows, attend):
  """The block on rows [T, D] through the operators' public calls; `attend` makes attention rows of q, k, v [T, H, hd]."""
  D, H, hd = block.hidden_dim, block.num_heads, block.head_dim
  P = dict(block.named_parameters())
  w = recml_amd.quantize_rows(torch.cat([P[n + "_kernel"].reshape(D, H * hd) for n in "uqkv"], 1).t())
  w_out = recml_amd.quantize_rows(P["output_kernel"].reshape(H * hd, D).t())
  bias = torch.cat([P[n + "_bias"].reshape(-1) for n in "uqkv"]) if block.use_bias else None
  normed = recml_amd.norm_rows8(rows, P["input_ln_gamma"], P["input_ln_beta"], block.eps)
  uqkv = recml_amd.gemm_rows8(normed, w, bias, True, dtype=rows.dtype).view(-1, 4, H, hd)
  u, q, k, v = uqkv.unbind(1)
  gated = recml_amd.norm_rows8(attend(q, k, v).reshape(-1, H * hd), P["attn_ln_gamma"].reshape(-1), P["attn_ln_beta"].reshape(-1), block.eps, gate=u.reshape(-1, H * hd))
  return recml_amd.gemm_rows8(gated, w_out, P["output_bias"] if block.use_bias else None, residual=rows, dtype=rows.dtype)


@pytest.mark.parametrize("use_bias", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_block_is_the_run_of_its_operators(gpu, dtype, use_bias):
  block = _model(dtype, D=136, H=1 if dtype == F32 else 17, use_bias=use_bias).decoder_blocks[0]
  H, hd, D, L = block.num_heads, block.head_dim, 136, 40
  lens = torch.tensor([40, 7, 0, 33], dtype=torch.int32, device=gpu)
  offsets = torch.tensor([0, 40, 47, 47, 80], dtype=torch.int32, device=gpu)
  x = torch.randn((4, L, D), generator=_gen(1)).to(dtype).to(gpu)
  pos = (torch.randn((H, 2 * L - 1), generator=_gen(2)) * 0.1).to(gpu)
  block.quantize()
  got = block(x, seq_lens=lens, pos_bias=pos)
  to4 = lambda t: t.reshape(4, L, H, hd)
  want = _by_hand(block, x.reshape(-1, D), lambda q, k, v: recml_amd.hstu_attention(to4(q), to4(k), to4(v), seq_lens=lens, n=float(L), pos_bias=pos))
  assert torch.equal(got.reshape(-1, D), want)
  packed = torch.cat([x[b, : int(n)] for b, n in enumerate(lens.tolist())])
  got = block.forward_jagged(packed, offsets, L, pos_bias=pos)
  want = _by_hand(block, packed, lambda q, k, v: recml_amd.hstu_attention(q, k, v, seq_offsets=offsets, max_len=L, n=float(L), pos_bias=pos))
  assert torch.equal(got, want)
  mask = torch.tril(torch.ones((L, L), dtype=torch.bool, device=gpu)).expand(4, L, L).contiguous()
  got = block(x, attention_mask=mask)
  want = _by_hand(block, x.reshape(-1, D), lambda q, k, v: recml_amd.pointwise_attention(to4(q), to4(k), to4(v), mask, None))
  assert torch.equal(got.reshape(-1, D), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_block_over_the_cache_is_the_run_of_its_operators(gpu, dtype):
  model = _model(dtype)
  model.quantize()
  block, B, L, n = model.decoder_blocks[0], 3, 50, 2
  cache = model.new_cache(B, L, bits=8, page_size=32)
  old = (torch.randn((B, L, 2, 32), generator=_gen(1)) * 0.4).to(gpu)
  starts = torch.tensor([0, 31, 48], dtype=torch.int32, device=gpu)
  recml_amd.kv_write(cache.layers[0], old, old.flip(1), cache.page_table, torch.zeros_like(starts))
  x = torch.randn((B, n, 64), generator=_gen(2)).to(dtype).to(gpu)

  def attend(q, k, v):
    to4 = lambda t: t.reshape(B, n, 2, 32)
    recml_amd.kv_write(cache.layers[0], to4(k), to4(v), cache.page_table, starts)
    return recml_amd.cached_attention(to4(q), cache.layers[0], cache.page_table, starts + n, max_len=L)

  got = block.forward_cached(x, cache.layers[0], cache.page_table, starts + n, starts, L)
  assert torch.equal(got.reshape(-1, 64), _by_hand(block, x.reshape(-1, 64), attend))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_8_bits_stand_for_the_model(gpu, dtype):
  """A model's outputs beside its own in its parameters' type.  A value of 8 bits is off by at most 2^-4 of itself, uniformly: 2^-4 / sqrt(3)
  in the mean square, so a product of two by 0.051 of the square root of the sum of its terms' squares.  A block has two such products one
  behind the other beside a residual that is exact: 0.051 of what it adds for each, and for the attention's logits and values between
  them; two blocks and the head (0.051 again): under 0.051 * (2 * 4 + 1)."""
  model = _model(dtype)
  ids, lens = torch.randint(0, 300, (5, 40), generator=_gen(5)).to(gpu), torch.tensor([40, 3, 17, 1, 25], dtype=torch.int32, device=gpu)
  plain = model(ids, seq_lens=lens, jagged=True).double()
  for head in (False, True):
    model.quantize(head=head)
    for jagged in (True, False):
      got = model(ids, seq_lens=lens, jagged=jagged).double()
      rows = torch.arange(40, device=gpu)[None, :] < lens[:, None]
      off = float((got - plain)[rows].norm() / plain[rows].norm())
      assert 1e-4 < off < 0.051 * 9, (head, jagged, off)
  model.dequantize()
  assert torch.equal(model(ids, seq_lens=lens, jagged=True).double(), plain)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_serving_in_8_bits(gpu, dtype):
  """prefill and extend go by the same weights: events one by one have the whole history's outputs, but for the cache's rounding and for codes
  that fall to the other side of a border.  (The cache's 8 bits are the rows' own kind of rounding, once more for keys and values.)"""
  model = _model(dtype)
  model.quantize(head=True)
  B, L = 4, 30
  ids, lens = torch.randint(0, 300, (B, L), generator=_gen(7)).to(gpu), torch.full((B,), L, dtype=torch.int32, device=gpu)
  want = model(ids, seq_lens=lens).double()
  cache = model.new_cache(B, L, bits=8)
  first = model.prefill(ids[:, :20], cache, seq_lens=torch.full((B,), 20, device=gpu)).double()
  rest = torch.cat([model.extend(ids[:, i : i + 2], cache) for i in range(20, L, 2)], 1).double()
  for got, part in ((first, want[:, :20]), (rest, want[:, 20:])):
    assert float((got - part).norm() / part.norm()) < 0.051 * 9
  assert int(cache.lengths.min()) == L


def test_a_step_captured_and_replayed(gpu):
  model = _model(BF16, D=128, H=2)
  model.quantize(head=True)
  B, L = 6, 64
  ids = torch.randint(0, 300, (B, 40), generator=_gen(8)).to(gpu)
  caches = [model.new_cache(B, L, bits=4) for _ in range(2)]
  for cache in caches:
    model.prefill(ids, cache, seq_lens=torch.full((B,), 40, device=gpu))
  new = torch.zeros((B, 1), dtype=torch.int64, device=gpu)
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    model.extend(new, model.new_cache(B, L, bits=4))
  side.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = model.extend(new, caches[0])
  for i in range(4):
    new.copy_(torch.randint(0, 300, (B, 1), generator=_gen(20 + i)).to(gpu))
    want = model.extend(new, caches[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want), i


def test_refused(gpu):
  model = _model(BF16)
  ids, lens = torch.zeros((2, 8), dtype=torch.int64, device=gpu), torch.tensor([8, 3], dtype=torch.int32, device=gpu)
  model.quantize(head=True)
  model.requires_grad_(True)
  with pytest.raises(ValueError, match="no gradient"):
    model(ids, seq_lens=lens)
  with pytest.raises(ValueError, match="no gradient"):
    model.log_probs(ids, ids, seq_lens=lens)
  with torch.no_grad():
    model(ids, seq_lens=lens)
  model.requires_grad_(False)
  model.load_state_dict(model.state_dict())
  with pytest.raises(ValueError, match="changed since quantize"):
    model(ids, seq_lens=lens)
  model.quantize(head=True)
  model(ids, seq_lens=lens)
  with torch.no_grad():
    model.reverse_embedding.mul_(2.0)
  with pytest.raises(ValueError, match="head's weight has changed"):
    model(ids, seq_lens=lens)
  model.quantize()
  model(ids, seq_lens=lens)
  with pytest.raises(ValueError, match="no output head"):
    _model(BF16, head=False).quantize(head=True)
  x = torch.zeros((2, 64), dtype=BF16, device=gpu, requires_grad=True)
  with pytest.raises(ValueError, match="no gradient"):
    recml_amd.quantize_rows(x)
  with pytest.raises(ValueError, match="no gradient"):
    recml_amd.norm_rows8(x.detach(), x[0])
  rows = recml_amd.quantize_rows(x.detach())
  with pytest.raises(ValueError, match="no gradient"):
    recml_amd.gemm_rows8(rows, rows, residual=x[:, :2])


def test_operators_refuse(gpu):
  x = torch.zeros((3, 64), dtype=BF16, device=gpu)
  rows = recml_amd.quantize_rows(x)
  for call, word in [
      (lambda: recml_amd.quantize_rows(x.half()), "dtype"), (lambda: recml_amd.quantize_rows(x[:, :0]), "W from 1"), (lambda: recml_amd.quantize_rows(x.sum()), "W from 1"),
      (lambda: recml_amd.norm_rows8(x, None), "gamma"), (lambda: recml_amd.norm_rows8(x, x[0].float()), "gamma must be"), (lambda: recml_amd.norm_rows8(x, x[0, :8]), "gamma must be"),
      (lambda: recml_amd.norm_rows8(x, x[0], x[0].cpu()), "beta must live"), (lambda: recml_amd.norm_rows8(x, x[0], gate=x[:2]), "gate must be"),
      (lambda: recml_amd.norm_rows8(x, x[0], add=x.float()), "add must be"), (lambda: rows.values(torch.float16), "dtype must be"),
      (lambda: recml_amd.gemm_rows8(rows, recml_amd.quantize_rows(x[:, :32])), "rows of 64"), (lambda: recml_amd.gemm_rows8(rows, rows, dtype=torch.float16), "dtype must be"),
      (lambda: recml_amd.gemm_rows8(rows, rows, x[0]), "bias must be"), (lambda: recml_amd.gemm_rows8(rows, rows, residual=x), "residual must be"),
      (lambda: recml_amd.gemm_rows8(rows, rows, x[0, :3].float()), "bias must be"), (lambda: recml_amd.Rows8(rows.codes, rows.exponents, 129), "codes"),
      (lambda: recml_amd.Rows8(rows.codes[:, :64], rows.exponents, 64), "contiguous"), (lambda: recml_amd.Rows8(rows.codes, rows.exponents[:, :2].contiguous(), 64), "exponents")]:
    with pytest.raises(ValueError, match=word):
      call()
  with pytest.raises(AttributeError):
    rows.width = 3


def test_copies_and_pickles(gpu):
  model = _model(BF16)
  model.quantize(head=True)
  ids, lens = torch.randint(0, 300, (2, 8), generator=_gen(1)).to(gpu), torch.tensor([8, 3], dtype=torch.int32, device=gpu)
  want = model(ids, seq_lens=lens)
  again = copy.deepcopy(model)
  again.quantize(head=True)
  assert torch.equal(again(ids, seq_lens=lens), want)
  rows = model.decoder_blocks[0]._rows8[0]
  file = io.BytesIO()
  torch.save(rows, file)
  file.seek(0)
  back = torch.load(file, weights_only=False)
  assert torch.equal(back.codes, rows.codes) and torch.equal(back.exponents, rows.exponents) and back.width == rows.width
  assert not any("rows8" in name for name in model.state_dict())
