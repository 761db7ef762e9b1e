"""Log probabilities of given tokens, entropy and the largest alternatives, and their gradient, against 64 bits."""

import math

import pytest
import torch

import recml_amd
from tests import serve_reference as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
STEP = 2.0**-24


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _logits(rows, vocab, dtype, seed, std=2.5):
  return (torch.randn((rows, vocab), generator=_gen(seed)) * std).to(dtype)


def _sums_off(vocab):
  """How far ln s may be off, in steps of 2^-24: a thread's 64 additions and a tree of them, exponents whose arguments are off by
  1.5 steps of their size (the sum of p |x - m| is at most ln V), the logarithm's own 4."""
  return (64 + math.log2(vocab + 1) + 4 + 3 * math.log(vocab + 1)) * STEP


def _check(got, x, tokens, top, entropy):
  want = R.log_probs(x, tokens if tokens is not None else torch.zeros((x.shape[0], 1), dtype=torch.int64), top)
  vocab = x.shape[1]
  span = torch.nan_to_num(x.double(), neginf=0, posinf=0).abs().amax() * 2
  tol = 2 * _sums_off(vocab) + 4 * STEP * (span + math.log(vocab + 1))
  def close(a, b, extra=0.0):
    a = a.cpu().double()
    assert a.shape == b.shape
    fine = torch.isfinite(b)
    assert torch.equal(fine, torch.isfinite(a)) and torch.equal(torch.isnan(a), torch.isnan(b))
    assert not fine.any() or float((a - b)[fine].abs().max()) <= tol + extra, (float((a - b)[fine].abs().max()), float(tol + extra))
  if tokens is not None:
    close(got.log_probs, want[0])
  if entropy:
    close(got.entropy, want[1], 4 * _sums_off(vocab) * math.log(vocab + 1))
  if top:
    assert torch.equal(got.top_tokens.cpu(), want[3])
    close(got.top_log_probs, want[2])


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 63), (7, 512), (3, 513), (2, 2047), (2, 4096), (3, 4097), (2, 8191), (5, 9001), (2, 16384), (1, 16391), (3, 20011),
          (1, 100003), (2, 300000)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward(gpu, rows, vocab, dtype):
  x = _logits(rows, vocab, dtype, vocab)
  tokens = torch.randint(0, vocab, (rows, 3), generator=_gen(1))
  for top in sorted({0, 1, min(5, vocab), min(64, vocab), min(100, vocab), min(256, vocab)}):
    _check(recml_amd.token_log_probs(x.cuda(), tokens.cuda(), top=top, entropy=True), x, tokens, top, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab,count,top", [(1, 1, 1, 0), (3, 2, 2, 1), (4, 8, 1, 3), (5, 63, 1, 0), (6, 4097, 5, 10), (3, 9001, 1, 64), (2, 20011, 100, 100), (1, 100003, 2, 256)])
def test_gradient(gpu, rows, vocab, count, top, dtype):
  x = _logits(rows, vocab, dtype, vocab + 1)
  tokens = torch.randint(0, vocab, (rows, count), generator=_gen(2))
  tokens[0, -1] = tokens[0, 0]                      # the same token twice
  if rows > 2:
    tokens[2] = -1                                  # a row that asks for nothing
  g = [torch.randn(s, generator=_gen(3 + i)) for i, s in enumerate([(rows, count), (rows,), (rows, top)])]
  for used in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
    if used[2] and not top:
      continue
    xs = x.cuda().requires_grad_(True)
    got = recml_amd.token_log_probs(xs, tokens.cuda(), top=top, entropy=True)
    outs = [(o, gg.cuda()) for o, gg, u in zip((got.log_probs, got.entropy, got.top_log_probs), g, used) if u]
    d = torch.autograd.grad([o for o, _ in outs], xs, [gg for _, gg in outs])[0].cpu()
    want = R.log_probs(x, tokens, top, *(gg if u else None for gg, u in zip(g, used)))
    lp, inner = want[5], want[6]
    p = lp.exp()
    # p is off by its exponent's error; the sum of gradients by its additions, the entropy's part by the entropy's error
    size = sum(gg.double().abs().reshape(rows, -1).sum(-1, keepdim=True) for gg, u in zip(g, used) if u)
    off = 8 * STEP * lp.abs().nan_to_num(posinf=0) + 3 * _sums_off(vocab)
    tol = p * (inner.abs() * off + size * (8 * _sums_off(vocab) * (1 + math.log(vocab + 1)))) + 4 * STEP * (size * p + want[4].abs()) + 1e-30
    tol = tol + torch.finfo(dtype).eps / 2 * want[4].abs()
    tol = tol + (STEP * (count + top) * size if max(count, top) > 1 else 0)
    if dtype == BF16:
      tol = tol + 2.0**-133 * 2                     # (values below bf16's smallest steps)
    bad = (d.double() - want[4]).abs() > tol
    assert d.dtype == dtype and not bad.any(), (used, float((d.double() - want[4]).abs().max()))
    if rows > 2 and used == (1, 0, 0):
      assert not d[2].any()


def test_gradient_against_differences(gpu):
  x = _logits(2, 41, F32, 5, 1.0).double()
  tokens = torch.tensor([[3, 3], [40, 0]])
  g = [torch.randn(s, generator=_gen(i)).double() for i, s in enumerate([(2, 2), (2,), (2, 4)])]
  xs = x.float().cuda().requires_grad_(True)
  got = recml_amd.token_log_probs(xs, tokens.cuda(), top=4, entropy=True)
  d = torch.autograd.grad([got.log_probs, got.entropy, got.top_log_probs], xs, [gg.float().cuda() for gg in g])[0].cpu().double()
  def loss(y):
    w = R.log_probs(y, tokens, 4)
    return (w[0] * g[0]).sum() + (w[1] * g[1]).sum() + (w[2] * g[2]).sum()
  h = 1e-5
  for r in range(2):
    for c in range(41):
      e = torch.zeros_like(x)
      e[r, c] = h
      assert abs(float(loss(x + e) - loss(x - e)) / (2 * h) - float(d[r, c])) < 1e-5     # (h^2 of third derivatives, fp32 sums)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [10, 700, 5000, 20000, 70001])
def test_ties_masked_and_odd_rows(gpu, vocab, dtype):
  """All equal; all but a few masked; nothing but -inf; NaN; +inf; falling and rising rows; zeros of either sign."""
  rows = [torch.zeros(vocab), torch.full((vocab,), -math.inf), torch.full((vocab,), -math.inf), _logits(1, vocab, F32, 3)[0], _logits(1, vocab, F32, 4)[0],
          torch.linspace(5, -5, vocab), torch.linspace(-5, 5, vocab), torch.where(torch.arange(vocab) % 2 == 0, -0.0, 0.0),
          torch.where(torch.arange(vocab) < vocab // 2, -math.inf, 1.0), _logits(1, vocab, F32, 6)[0]]
  rows[2][vocab - 1], rows[2][2] = 1.0, 1.0
  rows[3][vocab // 2] = math.nan
  rows[4][vocab // 3] = math.inf
  rows[9][::3] = -math.inf
  x = torch.stack(rows).to(dtype)
  tokens = torch.stack([torch.full((len(rows),), vocab - 1), torch.full((len(rows),), 2), torch.full((len(rows),), -5), torch.full((len(rows),), vocab)], 1)
  for top in (1, 7, 10):
    _check(recml_amd.token_log_probs(x.cuda(), tokens.cuda(), top=top, entropy=True), x, tokens, top, True)
  fine = [0, 2, 5, 6, 7, 8, 9]
  xs = x[fine].cuda().requires_grad_(True)
  tk = tokens[fine][:, [0, 2]]
  got = recml_amd.token_log_probs(xs, tk.cuda(), top=3, entropy=True)
  ge, gt = torch.randn(len(fine), generator=_gen(1)), torch.randn((len(fine), 3), generator=_gen(2))
  d = torch.autograd.grad([got.entropy, got.top_log_probs], xs, [ge.cuda(), gt.cuda()])[0].cpu()
  want = R.log_probs(x[fine], tk, 3, None, ge, gt)[4]
  assert (d.double() - want).abs().max() <= 2e-5 + torch.finfo(dtype).eps / 2 * want.abs().max()   # (fp32 sums of 1e-7 times gradients of up to 10)
  bad = x[[1, 3, 4]].cuda().requires_grad_(True)
  got = recml_amd.token_log_probs(bad, tokens[[1, 3, 4]][:, :1].cuda(), entropy=True)
  assert torch.isnan(torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), bad)[0]).all()
  past = x[:1].cuda().requires_grad_(True)
  assert torch.isnan(torch.autograd.grad(recml_amd.token_log_probs(past, tokens[:1, 3:].cuda()).log_probs.sum(), past)[0]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(gpu, dtype):
  """Rows that start anywhere, with gaps between them; leading axes; one token a row or several; nothing asked."""
  wide = _logits(12, 777, dtype, 9).cuda()
  for x in (wide[:, 3:700], wide[::2, 1:], wide.reshape(3, 4, 777)[:, 1:, 5:], wide.t()[:300], wide[5, 2:], wide[:1].expand(4, 777), wide[:0]):
    flat = x.reshape(-1, x.shape[-1])
    tokens = torch.randint(0, x.shape[-1], x.shape[:-1], generator=_gen(1))
    got = recml_amd.token_log_probs(x, tokens.cuda().to(torch.int32), top=4, entropy=True)
    assert got.log_probs.shape == x.shape[:-1] and got.top_tokens.shape == (*x.shape[:-1], 4)
    if flat.shape[0]:
      _check(recml_amd.TokenLogProbs(got.log_probs.reshape(-1, 1), got.entropy.reshape(-1), got.top_log_probs.reshape(-1, 4), got.top_tokens.reshape(-1, 4)),
             flat.cpu(), tokens.reshape(-1, 1), 4, True)
    leaf = wide.clone().requires_grad_(True)
    view = leaf[:, 3:700]
    d = torch.autograd.grad(recml_amd.token_log_probs(view, torch.full((12,), 2, device="cuda")).log_probs.sum(), leaf)[0]
    assert not d[:, :3].any() and not d[:, 700:].any()
    plain = view.detach().clone().requires_grad_(True)
    other = torch.autograd.grad(recml_amd.token_log_probs(plain, torch.full((12,), 2, device="cuda")).log_probs.sum(), plain)[0]
    # (not the same bits: where a row starts decides which thread adds what, so each ln s is off by its own _sums_off, p times that in the
    # gradient, p at most 1; then both round)
    tol = 2 * _sums_off(697) + 2 * STEP + torch.finfo(dtype).eps * other.double().abs()
    assert ((d[:, 3:700].double() - other.double()).abs() <= tol).all()
  got = recml_amd.token_log_probs(wide, None, entropy=True)
  assert got.log_probs is None and got.top_tokens is None
  assert recml_amd.token_log_probs(wide, torch.zeros((12, 0), dtype=torch.int64).cuda()).log_probs.shape == (12, 0)


def test_refusals(gpu):
  x = torch.zeros((4, 10), device="cuda")
  ids = torch.zeros(4, dtype=torch.int64, device="cuda")
  for bad, error in [((x.half(), ids), ValueError), ((x, ids.float()), ValueError), ((x, ids[:3]), ValueError), ((x.cpu(), ids.cpu()), ValueError), ((x, ids.cpu()), ValueError),
                     ((x,), ValueError), (([1.0], ids), TypeError), ((x[:, :0], ids), ValueError)]:
    with pytest.raises(error):
      recml_amd.token_log_probs(*bad)
  for top in (-1, 11, 257):
    with pytest.raises(ValueError):
      recml_amd.token_log_probs(x, ids, top=top)
  import torch.autograd.forward_ad as fwd
  with fwd.dual_level(), pytest.raises(Exception):
    recml_amd.token_log_probs(fwd.make_dual(x, x), ids)


def test_graph_replays_and_the_same_bits(gpu):
  x = _logits(5, 70001, BF16, 3).cuda()
  ids = torch.randint(0, 70001, (5, 2), generator=_gen(1)).cuda()
  g = torch.randn((5, 2), generator=_gen(2)).cuda()
  def step():
    leaf = x.detach().requires_grad_(True)
    got = recml_amd.token_log_probs(leaf, ids, top=9, entropy=True)
    return [got.log_probs.detach(), got.entropy.detach(), got.top_log_probs.detach(), got.top_tokens,
            torch.autograd.grad([got.log_probs, got.entropy], leaf, [g, g[:, 0].contiguous()])[0]]
  eager = step()
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    step()
  torch.cuda.current_stream().wait_stream(s)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    outs = step()
  for _ in range(3):
    for o in outs:
      o.zero_()
    graph.replay()
    again = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(eager, outs, again))


def test_the_python_way(gpu, monkeypatch):
  """What the native host side declines goes through the Python one: the same kernels, the same bits."""
  from recml_amd import _native
  x = _logits(6, 9001, BF16, 3).cuda()
  ids = torch.randint(0, 9001, (6, 2), generator=_gen(1)).cuda()
  def step():
    leaf = x.detach().requires_grad_(True)
    got = recml_amd.token_log_probs(leaf, ids, top=9, entropy=True)
    return [got.log_probs.detach(), got.entropy.detach(), got.top_log_probs.detach(), got.top_tokens,
            *(torch.autograd.grad(o.sum(), leaf, retain_graph=True)[0] for o in got[:3])]
  native = step()
  monkeypatch.setattr(_native, "token_log_probs", lambda *a: None)
  assert all(torch.equal(a, b) for a, b in zip(native, step()))


def test_second_derivatives(gpu):
  """The gradient's own gradient, in torch's steps behind the native node, against 64 bits."""
  x = _logits(3, 50, F32, 5, 1.0)
  x[0, ::4] = -math.inf
  ids = torch.tensor([[3, 3], [49, 1], [-1, 7]])
  w = torch.randn((3, 50), generator=_gen(2))
  def second(leaf, lp, ent, top):
    g = torch.autograd.grad((lp * lp).sum() + (ent * ent).sum() + top.square().sum(), leaf, create_graph=True)[0]
    return torch.autograd.grad((g * w.to(g)).sum(), leaf)[0]
  a = x.cuda().requires_grad_(True)
  got = recml_amd.token_log_probs(a, ids.cuda(), top=3, entropy=True)
  mine = second(a, got.log_probs, got.entropy, got.top_log_probs)
  b = x.double().requires_grad_(True)
  lp = torch.log_softmax(b, -1)
  masked = torch.isinf(x)
  safe = torch.where(masked, 0.0, lp)
  picked = torch.where(ids < 0, 0.0, lp.gather(1, ids.clamp(min=0)))
  ref = second(b, picked, -(lp.exp() * safe).sum(-1), lp.gather(1, got.top_tokens.cpu()))
  assert (mine.cpu().double() - ref).abs().max() <= 1e-4        # (fp32 sums of 50 terms, two derivatives of values up to 10)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [300, 4000, 16000, 40000])
def test_many_alternatives_and_many_ties(gpu, vocab, dtype):
  """Rows of a few values only: more entries reach the bound than the lists hold, and the lowest indices win."""
  few = torch.randint(0, 3, (4, vocab), generator=_gen(1)).float()
  few[1] = torch.where(torch.rand(vocab, generator=_gen(2)) < 0.9, 1.0, few[1])
  few[2, : vocab // 2] = -math.inf
  few[3] = -math.inf
  few[3, vocab // 2 :: 7] = -2.0
  x = few.to(dtype)
  tokens = torch.randint(0, vocab, (4, 1), generator=_gen(3))
  for top in (1, 16, 17, 64, 65, 200, 256):
    _check(recml_amd.token_log_probs(x.cuda(), tokens.cuda(), top=top), x, tokens, top, False)


def test_logits_past_four_billion_entries(gpu):
  """A last row whose entries lie past 2^32."""
  rows, vocab = 4300, 1_000_003
  x = torch.zeros((rows, vocab), dtype=BF16, device="cuda")
  last = _logits(1, vocab, BF16, 5)
  x[-1] = last[0].cuda()
  ids = torch.zeros((rows, 2), dtype=torch.int64, device="cuda")
  ids[-1, 1] = vocab - 1
  leaf = x.requires_grad_(True)
  got = recml_amd.token_log_probs(leaf, ids, top=4, entropy=True)
  _check(recml_amd.TokenLogProbs(*(t[-1:].detach() for t in got)), last, ids[-1:].cpu(), 4, True)
  d = torch.autograd.grad(got.log_probs[-1].sum(), leaf)[0]
  want = R.log_probs(last, ids[-1:].cpu(), 0, torch.ones((1, 2)))[4]
  assert not d[-2].any() and (d[-1].cpu().double() - want[0]).abs().max() <= 2.0**-7 + 1e-5      # (a gradient of 1 in bf16: 2^-8 of it, twice)


def test_a_loss_that_asks_for_some_rows_only(gpu):
  """Gradients that arrive as views: expanded, strided, of some outputs only."""
  x = _logits(6, 3000, F32, 3).cuda().requires_grad_(True)
  ids = torch.randint(0, 3000, (6, 4), generator=_gen(1)).cuda()
  got = recml_amd.token_log_probs(x, ids, top=3, entropy=True)
  a = torch.autograd.grad(got.log_probs.mean(), x, retain_graph=True)[0]                          # (an expanded scalar)
  b = torch.autograd.grad(got.log_probs, x, torch.full((4, 6), 1 / 24, device="cuda").t(), retain_graph=True)[0]
  assert torch.equal(a, b)
  c = torch.autograd.grad(got.top_log_probs[2, 1] + got.entropy[5], x)[0]
  assert c[2].any() and c[5].any() and not c[[0, 1, 3, 4]].any()


def test_a_vocabulary_past_32_bits_is_refused_and_entropy_by_any_truth(gpu):
  x = torch.zeros((1, 1), device="cuda").expand(1, 2**32 + 8)           # (no memory behind it; refused before a copy is made)
  with pytest.raises(ValueError, match="V from 1"):
    recml_amd.token_log_probs(x, torch.zeros(1, dtype=torch.int64, device="cuda"))
  y, ids = torch.randn((3, 50), generator=_gen(1)).cuda(), torch.arange(3).cuda()
  want = recml_amd.token_log_probs(y, ids, entropy=True)
  got = recml_amd.token_log_probs(y, ids, entropy=1)
  assert torch.equal(got.entropy, want.entropy) and torch.equal(got.log_probs, want.log_probs)
  assert recml_amd.token_log_probs(y, ids, entropy=0).entropy is None


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_large_gradient_of_the_entropy_beside_masked_entries(gpu, dtype):
  """Masked entries get none of it, however large it is."""
  x = (torch.randn((2, 70), generator=_gen(3))).to(dtype)
  x[0, 5:30] = -math.inf
  x = x.cuda().requires_grad_(True)
  d = torch.autograd.grad(recml_amd.token_log_probs(x, entropy=True).entropy, x, torch.full((2,), 2.0**40).cuda())[0]
  one = torch.autograd.grad(recml_amd.token_log_probs(x, entropy=True).entropy, x, torch.ones(2).cuda())[0]
  assert torch.equal(d, one * 2.0**40) and not d[0, 5:30].any() and d.isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab,count,top", [(3, 29, 100, 5), (2, 300, 129, 0), (2, 300, 700, 16), (2, 700, 513, 50), (3, 9001, 1000, 50), (2, 20011, 1500, 100), (1, 5000, 3001, 256)])
def test_gradients_of_many_tokens(gpu, rows, vocab, count, top, dtype):
  """More tokens a row than a workgroup has threads and than it lists, many of them the same: each entry gets the sum of its own in their order."""
  x = _logits(rows, vocab, dtype, vocab + 3)
  tokens = torch.randint(-1, vocab, (rows, count), generator=_gen(2))
  tokens[:, 5:9] = tokens[:, 3:4]
  tokens[:, -1] = tokens[:, 3]
  g = [torch.randn(s, generator=_gen(3 + i)) for i, s in enumerate([(rows, count), (rows,), (rows, top)])]
  xs = x.cuda().requires_grad_(True)
  def run():
    got = recml_amd.token_log_probs(xs, tokens.cuda(), top=top, entropy=True)
    return torch.autograd.grad([got.log_probs, got.entropy] + ([got.top_log_probs] if top else []), xs, [t.cuda() for t in g[: 3 if top else 2]])[0].cpu()
  d = run()
  assert torch.equal(d, run())
  want = R.log_probs(x, tokens, top, *(g if top else g[:2]))
  lp, inner = want[5], want[6]
  p = lp.exp()
  # an entry's own gradients: as many roundings of partial sums up to their size as it has; the rest as in test_gradient
  size = sum(t.double().abs().reshape(rows, -1).sum(-1, keepdim=True) for t in g)
  off = 8 * STEP * lp.abs().nan_to_num(posinf=0) + 3 * _sums_off(vocab)
  tol = p * (inner.abs() * off + size * (8 * _sums_off(vocab) * (1 + math.log(vocab + 1)))) + 4 * STEP * (size * p + want[4].abs()) + 2.0**-132
  tol = tol + torch.finfo(dtype).eps / 2 * want[4].abs() + STEP * (count + top) * size * p
  ids = tokens.clamp(min=0)
  mine = torch.zeros((rows, vocab), dtype=torch.float64)
  mine.scatter_add_(1, ids, g[0].double().abs() * (tokens >= 0))
  times = torch.zeros((rows, vocab), dtype=torch.float64).scatter_add_(1, ids, (tokens >= 0).double())
  if top:
    mine.scatter_add_(1, want[3], g[2].double().abs())
    times.scatter_add_(1, want[3], torch.ones_like(g[2].double()))
  tol = tol + STEP * times * mine
  bad = (d.double() - want[4]).abs() > tol
  assert not bad.any(), (float((d.double() - want[4]).abs().max()), int(bad.sum()))


def test_a_captured_backward_beside_an_eager_graph_is_refused(gpu):
  """The leaves' accumulators of an eager graph that lives belong to a stream that is not captured.  Refused before the engine meets it,
  through the operator's own leaf and through one further up; without the eager graph the same step is captured and replayed."""
  ids = torch.tensor([3, 4, 5]).cuda()
  h = torch.randn((3, 16), generator=_gen(1)).cuda()
  w = (torch.randn((16, 40), generator=_gen(2))).cuda().requires_grad_(True)
  x = torch.randn((3, 40), generator=_gen(3)).cuda().requires_grad_(True)
  one = torch.ones(3).cuda()
  for leaf, logits in ((x, lambda: x), (w, lambda: h @ w)):
    def step():
      return torch.autograd.grad(recml_amd.token_log_probs(logits(), ids).log_probs, leaf, one)[0]
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
      step()
    torch.cuda.current_stream().wait_stream(s)
    lives = recml_amd.token_log_probs(logits(), ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      h.clone()
      with pytest.raises(ValueError, match="eager graph"):
        recml_amd.token_log_probs(logits(), ids)
      with torch.no_grad():
        recml_amd.token_log_probs(logits(), ids)
    del lives, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      got = step()
    for _ in range(3):
      got.zero_()
      graph.replay()
      assert torch.equal(step(), want)
      torch.cuda.synchronize()
      assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(2, 700), (1100, 700), (2, 3001), (2, 40000)])
def test_rows_of_one_value(gpu, rows, vocab, dtype):
  """Everything ties: the lowest tokens, after the two that are larger; negative values, zeros of both signs, -inf and NaN."""
  for value in (0.0, -0.0, -1.5, 2.75, -math.inf, math.nan):
    x = torch.full((rows, vocab), value, dtype=dtype)
    if value == value:
      x[:, 650], x[:, 333] = 3.0, 4.0
    got = recml_amd.token_log_probs(x.cuda(), top=20)
    want = [333, 650, *range(18)] if value == value else list(range(20))
    assert torch.equal(got.top_tokens.cpu(), torch.tensor(want).expand(rows, 20)), value
    assert bool(got.top_log_probs.isnan().all()) == (value != value)


@pytest.mark.parametrize("rows,vocab", [(3, 70), (1100, 90), (2, 40000)])
def test_statistics_without_the_entropy(gpu, rows, vocab):
  """From C: a forward without an entropy serves a backward without its gradient; one with it is told so by NaN, never by another number."""
  import ctypes as C
  from recml_amd import _lib_serve
  lib = _lib_serve.load()
  x = _logits(rows, vocab, F32, 3).cuda()
  ids = torch.randint(0, vocab, (rows, 1), generator=_gen(1)).cuda()
  ones = torch.ones(rows).cuda()
  def run(entropy, g_tokens, g_entropy):
    lp, ent, stats, d = torch.empty(rows).cuda(), torch.empty(rows).cuda(), torch.full((rows, 3), 7.0).cuda(), torch.full((rows, vocab), 7.0).cuda()
    a = _lib_serve.HstuLogProbsArgs()
    a.struct_size, a.version = C.sizeof(a), _lib_serve.ABI_VERSION
    a.logits, a.rows, a.stride, a.vocab, a.dtype, a.count = x.data_ptr(), rows, vocab, vocab, _lib_serve.FP32, 1
    a.tokens, a.log_probs, a.stats, a.entropy = ids.data_ptr(), lp.data_ptr(), stats.data_ptr(), ent.data_ptr() if entropy else None
    work = torch.empty(max(16, lib.hstu_log_probs_workspace_bytes(C.byref(a))), dtype=torch.uint8).cuda()
    a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.hstu_log_probs_fwd(C.byref(a), stream) == 0
    a.d_logits, a.d_stride = d.data_ptr(), vocab
    a.g_tokens, a.g_entropy = ones.data_ptr() if g_tokens else None, ones.data_ptr() if g_entropy else None
    assert lib.hstu_log_probs_bwd(C.byref(a), stream) == 0
    torch.cuda.synchronize()
    return d
  xs = x.clone().requires_grad_(True)
  got = recml_amd.token_log_probs(xs, ids, entropy=True)
  plain = torch.autograd.grad(got.log_probs, xs, torch.ones_like(got.log_probs), retain_graph=True)[0]
  both = torch.autograd.grad([got.log_probs, got.entropy], xs, [torch.ones_like(got.log_probs), ones])[0]
  assert torch.equal(run(False, True, False), plain) and torch.equal(run(True, True, False), plain)
  assert torch.equal(run(True, True, True), both)
  assert run(False, True, True).isnan().all() and run(False, False, True).isnan().all()
