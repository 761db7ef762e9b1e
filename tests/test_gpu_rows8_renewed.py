"""HSTU's weights in 8 bits made again: captured calls go on with the new ones, and nothing else does with the old ones."""

import copy

import pytest
import torch

import recml_amd

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _model(dtype=BF16, seed=3, D=128, H=2, vocab=300):
  m = recml_amd.HSTU(vocab_size=vocab, max_positions=64, model_dim=D, num_heads=H, num_layers=2, dtype=dtype, device="cuda:0", seed=seed)
  m.decoder_blocks = torch.nn.ModuleList(recml_amd.HSTUBlock(D, H, use_bias=i == 1, dtype=dtype, device="cuda:0", generator=_gen(seed + i)) for i in range(2))
  g = _gen(seed + 1)
  with torch.no_grad():
    for p in m.parameters():
      p.add_((torch.randn(p.shape, generator=g) * 0.05).to(p))
  return m.eval()


def _places(model):
  rows = [r for block in model.decoder_blocks for r in (block._rows8[0], block._rows8[2])] + [model._head8[0]]
  return [t.data_ptr() for r in rows for t in (r.codes, r.exponents)] + [model.decoder_blocks[1]._rows8[1].data_ptr()]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inference", [False, True])
def test_a_captured_step_has_the_new_weights(gpu, dtype, inference):
  """Weights loaded and quantised again between replays, with other work on the memory in between."""
  model = _model(dtype)
  with torch.inference_mode(inference):
    model.quantize(head=True)
  B, L = 5, 64
  ids = torch.randint(0, 300, (B, 30), generator=_gen(8)).to(gpu)
  caches = [model.new_cache(B, L, bits=8) for _ in range(2)]
  for cache in caches:
    model.prefill(ids, cache, seq_lens=torch.full((B,), 30, device=gpu))
  new = torch.zeros((B, 1), dtype=torch.int64, device=gpu)
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    model.extend(new, model.new_cache(B, L, bits=8))
  side.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = model.extend(new, caches[0])
  places, before = _places(model), None
  for i in range(5):
    if i % 2:
      model.load_state_dict(_model(dtype, seed=20 + i).state_dict())
      model.quantize(head=True)
      noise = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=gpu) for _ in range(8)]      # (where freed codes would have lain)
      del noise
    assert _places(model) == places
    new.copy_(torch.randint(0, 300, (B, 1), generator=_gen(20 + i)).to(gpu))
    want = model.extend(new, caches[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want), i
    assert before is None or not torch.equal(out, before)
    before = out.clone()


def test_made_again_is_what_a_first_time_makes(gpu):
  model, other = _model(), _model(seed=9)
  model.quantize(head=True)
  model.load_state_dict(other.state_dict())
  model.quantize(head=True)
  other.quantize(head=True)
  for a, b in zip(model.decoder_blocks, other.decoder_blocks):
    for i in (0, 2):
      assert torch.equal(a._rows8[i].codes, b._rows8[i].codes) and torch.equal(a._rows8[i].exponents, b._rows8[i].exponents)
    assert (a._rows8[1] is None and b._rows8[1] is None) or torch.equal(a._rows8[1], b._rows8[1])
  assert torch.equal(model._head8[0].codes, other._head8[0].codes)
  ids, lens = torch.randint(0, 300, (3, 20), generator=_gen(1)).to(gpu), torch.tensor([20, 3, 11], dtype=torch.int32, device=gpu)
  assert torch.equal(model(ids, seq_lens=lens), other(ids, seq_lens=lens))


def _fresh_answer(block, x, lens):
  """What the block answers with codes that were never anybody's."""
  block = copy.deepcopy(block)
  block.dequantize()
  block.quantize()
  return block(x, seq_lens=lens)


def test_codes_are_not_written_under_another_block(gpu):
  """A shallow copy with parameters of its own shares the codes: once they are made again for one, the other is refused.  A deep copy has its own."""
  block = _model().decoder_blocks[1]
  block.quantize()
  deep, again = copy.deepcopy(block), copy.copy(block)
  x, lens = torch.randn((2, 8, 128), generator=_gen(1)).to(BF16).to(gpu), torch.tensor([8, 3], dtype=torch.int32, device=gpu)
  want = block(x, seq_lens=lens)
  again._parameters = dict(again._parameters)
  again.u_kernel = torch.nn.Parameter(block.u_kernel.detach() * 2, requires_grad=False)
  again.quantize()
  with pytest.raises(ValueError, match="changed since quantize"):
    block(x, seq_lens=lens)
  assert torch.equal(deep(x, seq_lens=lens), want)
  block.quantize()
  assert torch.equal(block(x, seq_lens=lens), want)
  assert torch.equal(again(x, seq_lens=lens), _fresh_answer(again, x, lens)) and not torch.equal(again(x, seq_lens=lens), want)


def test_converted_and_quantised_again(gpu):
  model, ids, lens = _model(F32), torch.randint(0, 300, (3, 20), generator=_gen(1)).to(gpu), torch.tensor([20, 3, 11], dtype=torch.int32, device=gpu)
  model.quantize(head=True)
  model(ids, seq_lens=lens)
  model.to(BF16)
  with pytest.raises(ValueError, match="changed since quantize"):
    model(ids, seq_lens=lens)
  model.quantize(head=True)
  other = _model(F32).to(BF16)
  other.quantize(head=True)
  assert torch.equal(model(ids, seq_lens=lens), other(ids, seq_lens=lens))


@pytest.mark.parametrize("loads", [0, 1])
def test_a_copy_answers_as_what_it_is_of(gpu, loads):
  """Bit for bit, and not with the old weights once it has others."""
  model, ids, lens = _model(), torch.randint(0, 300, (3, 20), generator=_gen(1)).to(gpu), torch.tensor([20, 3, 11], dtype=torch.int32, device=gpu)
  for i in range(loads):
    model.load_state_dict(_model(seed=30 + i).state_dict())
  model.quantize(head=True)
  want = model(ids, seq_lens=lens)
  again = copy.deepcopy(model)
  assert torch.equal(again(ids, seq_lens=lens), want)
  again.load_state_dict(_model(seed=40).state_dict())
  with pytest.raises(ValueError, match="changed since quantize"):
    again(ids, seq_lens=lens)
  assert torch.equal(model(ids, seq_lens=lens), want)
