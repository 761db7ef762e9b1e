"""Rows in 8 bits: calls of as many rows as a launch has threads for."""

import pytest
import torch

import recml_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normed", [False, True])
def test_a_table_of_many_narrow_rows(gpu, normed):
  """70 million rows of 64, eight threads each."""
  rows, width = 70_000_000, 64
  x = torch.zeros((rows, width), dtype=torch.bfloat16, device=gpu)
  tail = torch.randn((300, width), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
  x[-300:] = tail
  gamma = torch.full((width,), 1.5, dtype=torch.bfloat16, device=gpu)
  call = (lambda t: recml_amd.norm_rows8(t, gamma)) if normed else recml_amd.quantize_rows
  got, want = call(x), call(tail)
  del x
  assert torch.equal(got.codes[-300:], want.codes) and torch.equal(got.exponents[:, -300:], want.exponents)
  assert not got.codes[:-300].any() and (got.exponents[:, :-300] == 1).all()
  assert torch.equal(got.values()[-300:], want.values())
