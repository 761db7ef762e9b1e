"""Rows in 8 bits, and a model that keeps some, loaded where there is no GPU (map_location="cpu"): they load, and say what they cannot do."""

import copy
import io

import pytest
import torch

import recml_amd
from recml_amd import hstu_rows8


def _rows():
  return hstu_rows8.Rows8._of(torch.full((3, 128), 56, dtype=torch.uint8), torch.full((1, 3, 4), 127, dtype=torch.uint8), 100)


def _loaded(what):
  file = io.BytesIO()
  torch.save(what, file)
  file.seek(0)
  return torch.load(file, map_location="cpu", weights_only=False)


@pytest.mark.parametrize("again", [copy.deepcopy, _loaded])
def test_rows_without_a_gpu(again):
  rows = again(_rows())
  assert torch.equal(rows.codes, _rows().codes) and torch.equal(rows.exponents, _rows().exponents) and (rows.rows, rows.width) == (3, 100)
  for call in (lambda: rows.values(), lambda: rows.values(torch.float32), lambda: recml_amd.gemm_rows8(rows, rows), lambda: recml_amd.gemm_rows8(rows, rows, dtype=torch.float32)):
    with pytest.raises(ValueError, match="no CPU path"):
      call()
  with pytest.raises(ValueError, match="no CPU path"):
    hstu_rows8.Rows8(rows.codes, rows.exponents, rows.width)


def test_a_model_without_a_gpu(monkeypatch):
  model = recml_amd.HSTU(vocab_size=3, max_positions=8, model_dim=8, num_heads=2, num_layers=2, dtype=torch.float32).eval()
  monkeypatch.setattr(hstu_rows8, "quantize_rows", lambda x: _rows())
  model.quantize(head=True)
  monkeypatch.undo()
  again = _loaded(model)
  ids, lens = torch.zeros((2, 4), dtype=torch.int64), torch.tensor([4, 2], dtype=torch.int32)
  with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
    again(ids, seq_lens=lens)
  again.dequantize()
  assert all(torch.equal(a, b) for a, b in zip(again.parameters(), model.parameters()))
