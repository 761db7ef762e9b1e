"""Weights kept in 8 bits know whether they still are the parameters': written to, replaced, copied, saved and loaded.  (No GPU: what stands for
the rows in 8 bits here is a copy of the weight, and no block is run.)"""

import copy
import io

import pytest
import torch
from torch.nn.utils import parametrize, prune

import recml_amd
from recml_amd import hstu_rows8


@pytest.fixture
def stand_ins(monkeypatch):
  monkeypatch.setattr(hstu_rows8, "quantize_rows", lambda x: x.clone())
  monkeypatch.setattr(hstu_rows8, "gemm_rows8", lambda x, w, *args, **kw: x @ w.t())
  monkeypatch.setattr(torch.Tensor, "rows", property(lambda t: t.shape[0]), raising=False)


def _model(seed, dtype=torch.float32):
  return recml_amd.HSTU(vocab_size=11, max_positions=8, model_dim=8, num_heads=2, num_layers=2, dtype=dtype, seed=seed).eval()


def _saved(model):
  file = io.BytesIO()
  torch.save(model, file)
  file.seek(0)
  return torch.load(file, weights_only=False)


COPIES = {"deepcopy": copy.deepcopy, "saved and loaded": _saved}


def _runs(model):
  """Asks the blocks and the head as their calls do."""
  for block in model.decoder_blocks:
    block._check_rows8()
  if model._head8 is not None:
    x = torch.ones((2, model.model_dim), dtype=model.reverse_embedding.dtype)
    assert torch.equal(model._head(x), x @ model.reverse_embedding)


def _refused(model):
  for block in model.decoder_blocks:
    with pytest.raises(ValueError, match="changed since quantize"):
      block._check_rows8()
  if model._head8 is not None:
    with pytest.raises(ValueError, match="head's weight has changed"):
      model._head(torch.ones((2, model.model_dim), dtype=model.reverse_embedding.dtype))


@pytest.mark.parametrize("how", sorted(COPIES))
@pytest.mark.parametrize("loads", [0, 1, 2])
def test_a_copy_is_as_good_as_what_it_is_of(stand_ins, loads, how):
  model = _model(1)
  for i in range(loads):
    model.load_state_dict(_model(2 + i).state_dict())
  model.quantize(head=True)
  again = COPIES[how](model)
  _runs(again)
  assert torch.equal(again.decoder_blocks[1]._rows8[0], model.decoder_blocks[1]._rows8[0])
  _runs(COPIES[how](again))
  _runs(model)


@pytest.mark.parametrize("how", sorted(COPIES))
@pytest.mark.parametrize("before", [0, 1, 2])
@pytest.mark.parametrize("after", [1, 2])
def test_a_copy_notices_what_is_written_to_it(stand_ins, before, after, how):
  """However many times it was written to before it was copied."""
  model = _model(1)
  for i in range(before):
    model.load_state_dict(_model(2 + i).state_dict())
  model.quantize(head=True)
  again = COPIES[how](model)
  for i in range(after):
    again.load_state_dict(_model(7 + i).state_dict())
  _refused(again)
  _runs(model)
  again.quantize(head=True)
  _runs(again)


@pytest.mark.parametrize("how", sorted(COPIES))
def test_a_copy_of_what_has_changed_is_refused_too(stand_ins, how):
  model = _model(1)
  model.quantize(head=True)
  model.load_state_dict(_model(2).state_dict())
  _refused(model)
  again = COPIES[how](model)
  _refused(again)
  _refused(COPIES[how](again))
  again.load_state_dict(_model(3).state_dict())
  _refused(again)
  again.quantize(head=True)
  _runs(again)


@pytest.mark.parametrize("how", sorted(COPIES))
def test_a_copy_of_what_was_replaced_is_refused_too(stand_ins, how):
  model = _model(1)
  model.quantize(head=True)
  for block in model.decoder_blocks:
    block.q_kernel = torch.nn.Parameter(block.q_kernel.detach().clone(), requires_grad=False)
  model.reverse_embedding = torch.nn.Parameter(model.reverse_embedding.detach().clone(), requires_grad=False)
  _refused(model)
  _refused(COPIES[how](model))


def test_a_shallow_copy_sees_the_same_parameters(stand_ins):
  block = _model(1).decoder_blocks[0]
  block.quantize()
  again = copy.copy(block)
  again._check_rows8()
  with torch.no_grad():
    block.u_kernel.mul_(2.0)
  for b in (block, again):
    with pytest.raises(ValueError, match="changed since quantize"):
      b._check_rows8()


def test_parameters_that_do_not_count_their_writes_are_refused(stand_ins):
  """Those made under inference mode."""
  with torch.inference_mode():
    model = _model(1)
  with pytest.raises(ValueError, match="inference_mode"):
    model.quantize()
  with pytest.raises(ValueError, match="inference_mode"):
    model.decoder_blocks[0].quantize()
  assert all(block._rows8 is None for block in model.decoder_blocks)
  model = _model(1)
  model.reverse_embedding = None
  with torch.inference_mode():
    model.reverse_embedding = torch.nn.Parameter(torch.ones((8, 11)), requires_grad=False)
  with pytest.raises(ValueError, match="inference_mode"):
    model.quantize(head=True)
  assert all(block._rows8 is None for block in model.decoder_blocks)      # (before any work)


@pytest.mark.parametrize("how", sorted(COPIES))
def test_copies_made_under_inference_mode_are_refused(stand_ins, how):
  model = _model(1)
  model.quantize(head=True)
  with torch.inference_mode():
    again = COPIES[how](model)
  if any(p.is_inference() for p in again.parameters()):
    _refused(again)


def test_what_is_written_under_inference_mode_is_noticed(stand_ins):
  model = _model(1)
  with torch.inference_mode():
    model.quantize(head=True)
    _runs(model)
    model.load_state_dict(_model(2).state_dict())
    _refused(model)


def test_parameters_whose_memory_was_replaced_are_noticed(stand_ins):
  """Converted to another type or put elsewhere: the parameter stays, and its count too."""
  model = _model(1)
  model.quantize(head=True)
  model.to(torch.float32).to("cpu").eval().requires_grad_(False)
  _runs(model)
  model.to(torch.bfloat16)
  _refused(model)
  model.quantize(head=True)
  _runs(model)
  for p in model.parameters():
    p.data = p.data.clone()
  _refused(model)


def test_there_and_back_is_noticed(stand_ins):
  """Values that were rounded on the way may come to lie where the old ones lay."""
  for _ in range(20):
    model = _model(1)
    model.quantize(head=True)
    model.to(torch.bfloat16).to(torch.float32)
    _refused(model)


class _Scaled(torch.nn.Module):
  def __init__(self):
    super().__init__()
    self.scale = torch.nn.Parameter(torch.tensor(2.0), requires_grad=False)

  def forward(self, w):
    return w * self.scale


def test_what_parametrized_weights_are_made_of_is_noticed(stand_ins):
  """The tensor that is kept, and what its parametrization keeps."""
  block = _model(1).decoder_blocks[0]
  parametrize.register_parametrization(block, "u_kernel", _Scaled())
  made = block.parametrizations.u_kernel
  for change in (lambda: made.original.mul_(2.0), lambda: made[0].scale.add_(1.0), lambda: block.k_kernel.zero_()):
    block.quantize()
    assert torch.equal(block._rows8[0][: block.hidden_dim], (made.original * made[0].scale).reshape(block.hidden_dim, -1).t())
    block._check_rows8()
    again = copy.deepcopy(block)
    again._check_rows8()
    with torch.no_grad():
      change()
    with pytest.raises(ValueError, match="changed since quantize"):
      block._check_rows8()
    again._check_rows8()


def test_what_a_parametrized_head_is_made_of_is_noticed(stand_ins):
  model = _model(1)
  parametrize.register_parametrization(model, "reverse_embedding", _Scaled())
  model.quantize(head=True)
  _runs(model)
  with torch.no_grad():
    model.item_embedding.add_(1.0)
  _runs(model)
  with torch.no_grad():
    model.parametrizations.reverse_embedding.original.mul_(2.0)
  with pytest.raises(ValueError, match="head's weight has changed"):
    model._head(torch.ones((2, 8)))
  model.quantize(head=True)
  _runs(model)


def test_weights_that_a_hook_makes_are_refused(stand_ins):
  """A pruned weight is made again by the next forward only: what stands there may be old."""
  block = _model(1).decoder_blocks[0]
  prune.l1_unstructured(block, "output_kernel", amount=0.5)
  with pytest.raises(ValueError, match="output_kernel is a tensor that a hook makes"):
    block.quantize()
  prune.remove(block, "output_kernel")
  block.quantize()
  block._check_rows8()
  assert torch.equal(block._rows8[2], block.output_kernel.reshape(8, 8).t()) and int((block.output_kernel == 0).sum()) == 32
  prune.l1_unstructured(block, "u_kernel", amount=0.5)
  with pytest.raises(ValueError, match="u_kernel is a tensor that a hook makes"):
    block._check_rows8()


def test_what_is_not_quantised_may_change(stand_ins):
  """Norms and the output's bias are read as they are."""
  block = recml_amd.HSTUBlock(8, 2, use_bias=True)
  block.quantize()
  with torch.no_grad():
    for p in (block.input_ln_gamma, block.input_ln_beta, block.attn_ln_gamma, block.attn_ln_beta, block.output_bias):
      p.add_(1.0)
  block._check_rows8()
  with torch.no_grad():
    block.v_bias.add_(1.0)
  with pytest.raises(ValueError, match="changed since quantize"):
    block._check_rows8()


def test_a_call_that_fails_leaves_what_was_there(stand_ins, monkeypatch):
  """No memory, say: the codes stay where they lay, and are written by the next call."""
  model = _model(1)
  model.quantize(head=True)
  kept = [t.data_ptr() for block in model.decoder_blocks for t in (block._rows8[0], block._rows8[2])] + [model._head8[0].data_ptr()]
  model.load_state_dict(_model(2).state_dict())
  with monkeypatch.context() as m:
    calls = []

    def fails(x):
      calls.append(x)
      if len(calls) == 2:
        raise torch.OutOfMemoryError("none left")
      return x.clone()

    m.setattr(hstu_rows8, "quantize_rows", fails)
    with pytest.raises(torch.OutOfMemoryError):
      model.quantize(head=True)
  _refused(model)
  model.quantize(head=True)
  _runs(model)
  assert kept == [t.data_ptr() for block in model.decoder_blocks for t in (block._rows8[0], block._rows8[2])] + [model._head8[0].data_ptr()]
