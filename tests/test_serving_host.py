"""The native host side of the serving operators, where it can be looked at without a GPU."""

import pytest
import torch

from recml_amd import _native


def test_a_leafs_accumulator_outlives_the_walk_over_its_graph():
  """What a leaf without a graph of its own is asked for is made for the question, and has to be there until it is answered; the leaf of a graph
  that lives has the graph's."""
  x = torch.randn(3, requires_grad=True)
  assert _native.accumulators(x) == 1
  y = x * 2
  assert _native.accumulators(x) == 1 and _native.accumulators(y) == 1
  w = torch.randn(3, requires_grad=True)
  z = (y * w + x).sum() + w.exp().sum()
  assert _native.accumulators(z) == 2
  del y, z
  assert _native.accumulators(w) == 1
  assert _native.accumulators(torch.randn(3)) == 0 and _native.accumulators((x * w).detach()) == 0
  # (the walk leaves nothing behind and nothing out: gradients are what they were)
  (x * w).sum().backward()
  assert torch.equal(x.grad, w.detach()) and torch.equal(w.grad, x.detach())


def test_the_native_call_takes_what_it_reads():
  """A graph is made where the logits want a gradient: there is no argument for it."""
  x = torch.randn(2, 5)
  assert _native.token_log_probs(x, None, 1, False) is None           # (CPU tensors are for the Python side to refuse)
  for args in ((x, None, 1, False, True), (x, None, 1)):
    with pytest.raises(TypeError, match="4 arguments"):
      _native.token_log_probs(*args)
