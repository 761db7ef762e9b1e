"""The model's serving path: histories taken into a cache, new events run over it, items scored; and its loss."""

import math

import pytest
import torch

import recml_amd
from tests import serve_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _model(dtype, D=64, H=2, layers=2, vocab=300, positions=64, head=True, seed=3):
  m = recml_amd.HSTU(vocab_size=vocab, max_positions=positions, model_dim=D, num_heads=H, num_layers=layers, add_head=head, dtype=dtype, device="cuda:0", seed=seed,
                     scale_by_sqrt_dim=True)
  g = _gen(seed + 1)
  for p in m.parameters():                       # (weights of ones and zeros would hide what they scale)
    p.data.add_((torch.randn(p.shape, generator=g) * 0.05).to(p))
  return m.eval()


def _layer_norm(x, gamma, beta, eps):
  mean = x.mean(-1, keepdim=True)
  return (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps) * gamma + beta


def _block_reference(block, x, k_all, v_all, lengths, L, pos, ts, tab):
  """The block on the last rows x [B, n, D] of every history in 64 bits, over the kept keys and values [B, places, H, hd]."""
  P = {n: p.detach().cpu().double() for n, p in block.named_parameters()}
  y = _layer_norm(x, P["input_ln_gamma"], P["input_ln_beta"], block.eps)
  proj = lambda n: torch.nn.functional.silu(torch.einsum("bnd,dhe->bnhe", y, P[n + "_kernel"]))
  u, q, k, v = (proj(n) for n in "uqkv")
  out = []
  for b in range(x.shape[0]):
    held = torch.ones(k_all.shape[1], dtype=torch.bool)
    a, _, _ = R.attention(q[b], k_all[b], v_all[b], length=int(lengths[b]), max_len=L, held=held, pos_bias=pos, timestamps=None if ts is None else ts[b], ts_bias=tab)
    out.append(a)
  a = torch.stack(out).flatten(-2)
  a = _layer_norm(a, P["attn_ln_gamma"].flatten(), P["attn_ln_beta"].flatten(), block.eps) * u.flatten(-2)
  return torch.einsum("bnw,wd->bnd", a, P["output_kernel"].flatten(0, 1)) + x, k, v


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_block_over_the_cache(gpu, dtype, bits):
  """Rows of a block against 64 bits, over what the cache holds; and what it holds are the block's own keys and values, quantised."""
  model = _model(dtype)
  block, B, L, n = model.decoder_blocks[0], 3, 50, 2
  cache = model.new_cache(B, L, bits=bits, page_size=32)
  pages = cache.layers[0]
  old = (torch.randn((B, L, 2, 32), generator=_gen(1)) * 0.4).cuda()
  starts = torch.tensor([0, 31, 48], dtype=torch.int32).cuda()
  recml_amd.kv_write(pages, old, old.flip(1), cache.page_table, torch.zeros_like(starts))
  x = (torch.randn((B, n, 64), generator=_gen(2))).to(dtype)
  pos = torch.randn((2, 2 * L - 1), generator=_gen(3)) * 0.2
  ts = 1_600_000_000 + torch.randint(1, 10**5, (B, L), generator=_gen(4)).cumsum(1)
  tab = torch.randn((2, 129), generator=_gen(5)) * 0.2
  out = block.forward_cached(x.cuda(), pages, cache.page_table, starts + n, starts, L, pos_bias=pos.cuda(), timestamps=ts.cuda(), ts_bias=tab.cuda())
  k, v = (t.cpu().double() for t in recml_amd.kv_read(pages, cache.page_table, torch.zeros_like(starts), count=L, dtype=F32))
  want, wk, wv = _block_reference(block, x.double(), k, v, starts.cpu() + n, L, pos, ts, tab)
  # fp32: sums of up to 64 terms through two norms, whose 1/sigma (at most 30 here) carries their errors on.  bf16: the normed rows, the
  # projections, the attention and the gated rows each round once to 2^-8, of values of about 1, and go through products of 64 terms whose
  # weights have a 2-norm of about 1.
  assert (out.cpu().double() - want).norm() / want.norm() <= (1e-5 if dtype == F32 else 4 * 2.0**-8)
  for b in range(B):
    at = slice(int(starts[b]), int(starts[b]) + n)
    for kept, exact in ((k, wk), (v, wv)):
      # half a step of a code (2^-2 and 2^-4 of the value, or 1/4 and 2^-10 of the power), and the projection's own error
      size = exact[b].abs().amax(-1, keepdim=True)
      step = torch.maximum(exact[b].abs() * (0.25 if bits == 4 else 2.0**-4), size * (0.25 / 3.5 if bits == 4 else 2.0**-10 / 232))
      assert ((kept[b, at] - exact[b]).abs() <= step * 1.01 + size * (1e-5 if dtype == F32 else 3 * 2.0**-8)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_events_one_by_one_and_together(gpu, dtype):
  """The same events in one call, in several, packed or padded: each attends to the same places, so the results agree to the last bits
  of sums in another order.  (One layer: deeper ones would quantise rows that differ in those bits, and a code is 2^-4 of its value.)"""
  model = _model(dtype, layers=1)
  B, L, n = 3, 64, 6
  ids = torch.randint(1, 300, (B, 40 + n), generator=_gen(1)).cuda()
  ts = (1_600_000_000 + torch.randint(1, 10**5, (B, 40 + n), generator=_gen(2)).cumsum(1)).cuda()
  pos, tab = (torch.randn((2, 2 * L - 1), generator=_gen(3)) * 0.2).cuda(), (torch.randn((2, 129), generator=_gen(4)) * 0.2).cuda()
  lens = torch.tensor([40, 0, 17]).cuda()
  kw = dict(pos_bias=pos, ts_bias=tab)
  caches = [model.new_cache(B, L, bits=8, page_size=32, timestamps=True) for _ in range(3)]
  for c in caches:
    model.prefill(ids[:, :40], c, seq_lens=lens, timestamps=ts[:, :40], **kw)
    assert torch.equal(c.lengths.cpu(), lens.cpu().int())
  new, when = ids[:, 40:], ts[:, 40:]
  # (a row's time bias reads the next event's time: known for all but the last row of a call, so only calls that end with the event agree)
  together = model.extend(new, caches[0], timestamps=when, **kw)
  model.extend(new[:, : n - 1], caches[1], timestamps=when[:, : n - 1], **kw)
  last = model.extend(new[:, n - 1 :], caches[1], timestamps=when[:, n - 1 :], **kw)
  offsets = torch.arange(0, B * n + 1, n).cuda()
  packed = model.extend(new.reshape(-1), caches[2], offsets=offsets, max_new=n, timestamps=when.reshape(-1), **kw)
  for c in caches:
    assert torch.equal(c.lengths, caches[0].lengths) and torch.equal(c.timestamps, caches[0].timestamps)
  assert together.shape == (B, n, 300) and packed.shape == (B * n, 300)
  # bf16 results are rounded several times on the way; the roundings are the same but where fp32 sums differ in their last bits
  tol = 1e-5 if dtype == F32 else 4 * 2.0**-8
  close = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm()) <= tol
  assert close(packed.reshape(B, n, -1), together)
  assert close(last, together[:, n - 1 :])


def test_prefill_is_the_forward(gpu):
  """Whole histories attend to their own keys and values: the model's forward, its cache beside it."""
  for dtype in (F32, BF16):
    model = _model(dtype)
    ids = torch.randint(1, 300, (4, 50), generator=_gen(1)).cuda()
    lens = torch.tensor([50, 1, 0, 33]).cuda()
    pos = (torch.randn((99,), generator=_gen(3)) * 0.2).cuda()
    cache = model.new_cache(4, 50, bits=8, page_size=32)
    out = model.prefill(ids, cache, seq_lens=lens, pos_bias=pos)
    want = model(ids, seq_lens=lens, jagged=True, pos_bias=pos)
    # two runs of the same steps, rounded in other places: 2^-8 a step in bf16, sums in other orders in fp32
    assert (out.double() - want.double()).norm() / want.double().norm() <= (1e-5 if dtype == F32 else 8 * 2.0**-8)
    assert not out[2].any() and not out[3, 33:].any()


def test_kept_histories_stand_for_the_full_call(gpu):
  """With 8 bits the kept values are off by 2^-4 at most: the model's outputs for the last events come out near those of a call on all."""
  model = _model(F32)
  ids = torch.randint(1, 300, (3, 64), generator=_gen(1)).cuda()
  cache = model.new_cache(3, 64, bits=8, page_size=32)
  model.prefill(ids[:, :60], cache, seq_lens=torch.full((3,), 60).cuda())
  out = model.extend(ids[:, 60:], cache)
  full = model(ids, seq_lens=torch.full((3,), 64).cuda())[:, 60:]
  # keys and values each off by at most 2^-4 of themselves (and their block's smallest steps): 2 layers of 2 * 2^-4 before the residual
  assert (out - full).norm() / full.norm() <= 4 * 2.0**-4


def test_a_served_step_in_a_graph(gpu):
  """A step captured once and replayed as events come in: lengths, pages and times live on the GPU."""
  model = _model(BF16)
  pos, tab = (torch.randn((2, 127), generator=_gen(3)) * 0.2).cuda(), (torch.randn((2, 129), generator=_gen(4)) * 0.2).cuda()
  ids = torch.randint(1, 300, (2, 30), generator=_gen(1)).cuda()
  ts = (1_600_000_000 + torch.randint(1, 10**5, (2, 30), generator=_gen(2)).cumsum(1)).cuda()
  caches = [model.new_cache(2, 64, bits=4, page_size=32, timestamps=True) for _ in range(2)]
  for c in caches:
    model.prefill(ids[:, :20], c, seq_lens=torch.tensor([20, 7]).cuda(), timestamps=ts[:, :20], pos_bias=pos, ts_bias=tab)
  seen = torch.randint(1, 300, (2, 3), generator=_gen(7)).cuda()
  new, when = ids[:, :1].clone(), ts[:, :1].clone()
  def step(cache):
    logits = model.extend(new, cache, timestamps=when, pos_bias=pos, ts_bias=tab)
    got = recml_amd.token_log_probs(logits[:, -1], seen, top=5, entropy=True)
    return logits, *got
  step(caches[1])                                  # (warms up, then forgotten)
  caches[1].lengths.copy_(caches[0].lengths)
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    step(caches[1])
  torch.cuda.current_stream().wait_stream(s)
  caches[1].lengths.copy_(caches[0].lengths)
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g):
    outs = step(caches[1])
  caches[1].lengths.copy_(caches[0].lengths)
  for i in range(20, 26):
    new.copy_(ids[:, i : i + 1])
    when.copy_(ts[:, i : i + 1])
    g.replay()
    want = step(caches[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
  assert torch.equal(caches[0].lengths.cpu(), torch.tensor([26, 13], dtype=torch.int32))


def test_users_come_and_go_and_share_a_pool(gpu):
  """A pool of pages shared out by the caller: users without room lose what does not fit, the others never notice."""
  model = _model(F32, layers=1, head=False)
  ids = torch.randint(1, 300, (3, 40), generator=_gen(1)).cuda()
  table = torch.tensor([[4, -1], [0, 2], [-1, -1]], dtype=torch.int32).cuda()
  shared, own = model.new_cache(3, 64, bits=8, page_size=32, pages=5, page_table=table), model.new_cache(3, 64, bits=8, page_size=32)
  lens = torch.tensor([40, 40, 40]).cuda()
  for c in (shared, own):
    model.prefill(ids, c, seq_lens=lens)
  a, b = (model.extend(ids[:, :2], c) for c in (shared, own))
  assert torch.equal(a[1], b[1]) and not torch.equal(a[0], b[0]) and not torch.equal(a[2], b[2])
  own.reset(torch.tensor([0, 2]).cuda())
  assert own.lengths.tolist() == [0, 42, 0]
  fresh = model.new_cache(3, 64, bits=8, page_size=32)
  model.prefill(ids, fresh, seq_lens=torch.tensor([0, 40, 0]).cuda())
  model.extend(ids[1:2, :2].reshape(-1), fresh, offsets=torch.tensor([0, 0, 2, 2]).cuda(), max_new=2)
  assert torch.equal(model.extend(ids[:, 5:6], own), model.extend(ids[:, 5:6], fresh))


def test_the_loss_and_its_gradients(gpu):
  """log_probs over the model's head, trained: its gradients against torch's own steps on the same logits, and against differences."""
  model = _model(F32, vocab=97)
  model.requires_grad_(True)
  ids = torch.randint(1, 97, (3, 12), generator=_gen(1)).cuda()
  lens = torch.tensor([12, 5, 1]).cuda()
  nxt = torch.where(torch.arange(12, device="cuda")[None] < (lens - 1)[:, None], ids.roll(-1, 1), -1)
  def loss(got):
    return -(got.log_probs.sum() + 0.1 * got.entropy.sum()) / 15
  got = model.log_probs(ids, nxt, entropy=True, seq_lens=lens)
  assert got.log_probs.shape == (3, 12) and not got.log_probs[nxt < 0].any()
  ps = [p for p in model.parameters()]
  mine = torch.autograd.grad(loss(got), ps)
  lp = torch.log_softmax(model(ids, seq_lens=lens).double(), -1)
  picked = torch.where(nxt < 0, 0.0, lp.gather(-1, nxt.clamp(min=0)[..., None])[..., 0])
  plain = torch.autograd.grad(loss(recml_amd.TokenLogProbs(picked, -(lp.exp() * lp).sum(-1), None, None)), ps)
  for a, b in zip(mine, plain):
    assert (a.double() - b.double()).norm() <= 1e-4 * b.double().norm() + 1e-7         # (fp32 backwards of two layers on gradients that differ by 1e-6)
  # differences along a random direction of the head: the loss is smooth in it, third derivatives of about 1 times h^2
  w = model.reverse_embedding
  d = torch.randn(w.shape, generator=_gen(9)).cuda()
  i = [j for j, p in enumerate(ps) if p is w][0]
  h = 1e-2
  with torch.no_grad():
    ends = []
    for s in (h, -h):
      w.add_(s * d)
      ends.append(float(loss(model.log_probs(ids, nxt, entropy=True, seq_lens=lens)).double()))
      w.add_(-s * d)
  assert abs((ends[0] - ends[1]) / (2 * h) - float((mine[i] * d).sum())) <= 2e-3 * float(d.norm()) * float(mine[i].norm()) ** 0.5 + 1e-4


def test_what_serving_refuses(gpu):
  model = _model(F32, layers=1)
  cache = model.new_cache(2, 32)
  ids = torch.zeros((2, 1), dtype=torch.int64).cuda()
  with pytest.raises(ValueError):
    model.extend(ids[:1], cache)
  with pytest.raises(ValueError):
    model.extend(ids.reshape(-1), cache, offsets=torch.tensor([0, 1, 2]).cuda())
  with pytest.raises(ValueError):
    model.extend(ids, cache, timestamps=ids)
  with pytest.raises(ValueError):
    model.extend(ids, cache, timestamps=ids, ts_bias=torch.zeros(129).cuda())
  with pytest.raises(ValueError):
    model.prefill(torch.zeros((2, 33), dtype=torch.int64).cuda(), cache, seq_lens=torch.tensor([1, 1]).cuda())
  with pytest.raises(ValueError):
    _model(F32, layers=2).extend(ids, cache)
  with pytest.raises(ValueError):
    model.new_cache(2, 32, pages=4)
  with pytest.raises(ValueError, match="head"):
    _model(F32, head=False).log_probs(ids, ids, seq_lens=torch.tensor([1, 1]).cuda())
  dropped = recml_amd.HSTU(vocab_size=10, model_dim=32, num_heads=1, num_layers=1, dropout=0.5, device="cuda:0")
  with pytest.raises(ValueError, match="eval"):
    dropped.extend(ids, dropped.new_cache(2, 32))
  with pytest.raises(ValueError, match="head_dim"):
    recml_amd.HSTU(vocab_size=10, model_dim=40, num_heads=1, num_layers=1, device="cuda:0").new_cache(2, 32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_without_events(gpu, dtype):
  model = _model(dtype)
  cache = model.new_cache(2, 32)
  assert model.extend(torch.zeros((2, 0), dtype=torch.int64).cuda(), cache).shape == (2, 0, 300)
  none = torch.zeros(3, dtype=torch.int32).cuda()
  assert model.extend(torch.zeros(0, dtype=torch.int64).cuda(), cache, offsets=none, max_new=4).shape == (0, 300)
  out = model.prefill(torch.zeros((2, 5), dtype=torch.int64).cuda(), cache, seq_lens=torch.zeros(2, dtype=torch.int64).cuda())
  assert out.shape == (2, 5, 300) and not out.any() and cache.lengths.tolist() == [0, 0]


def test_packed_rows_of_no_user_and_past_max_new(gpu):
  """Rows before the first user's, behind the last one's and past `max_new` join no history: neither its length, nor its keys, nor its times."""
  model = _model(F32)
  pos, tab = (torch.randn((127,), generator=_gen(3)) * 0.2).cuda(), (torch.randn((129,), generator=_gen(4)) * 0.2).cuda()
  ids = torch.randint(1, 300, (2, 12), generator=_gen(1)).cuda()
  ts = (1_600_000_000 + torch.randint(1, 10**5, (2, 12), generator=_gen(2)).cumsum(1)).cuda()
  odd, plain = (model.new_cache(2, 64, bits=8, page_size=32, timestamps=True) for _ in range(2))
  for c in (odd, plain):
    model.prefill(ids[:, :6], c, seq_lens=torch.tensor([6, 4]).cuda(), timestamps=ts[:, :6], pos_bias=pos, ts_bias=tab)
  # user 0: rows 2 and 3; user 1: rows 4, 5 and 6, of which the third is past max_new; rows 0, 1, 7, 8: nobody's
  rows, when = torch.randint(1, 300, (9,), generator=_gen(5)).cuda(), (1_700_000_000 + torch.arange(9)).cuda()
  a = model.extend(rows, odd, offsets=torch.tensor([2, 4, 7]).cuda(), max_new=2, timestamps=when, pos_bias=pos, ts_bias=tab)
  b = model.extend(rows[2:6], plain, offsets=torch.tensor([0, 2, 4]).cuda(), max_new=2, timestamps=when[2:6], pos_bias=pos, ts_bias=tab)
  assert torch.equal(a[2:6], b)
  assert odd.lengths.tolist() == plain.lengths.tolist() == [8, 6]
  assert torch.equal(odd.timestamps, plain.timestamps)
  for x, y in zip(odd.layers, plain.layers):
    assert torch.equal(x.k, y.k) and torch.equal(x.v_scales, y.v_scales)
  step = dict(timestamps=ts[:, 6:7], pos_bias=pos, ts_bias=tab)
  assert torch.equal(model.extend(ids[:, 6:7], odd, **step), model.extend(ids[:, 6:7], plain, **step))


def test_times_of_another_shape_and_blocks_of_another_kind_are_refused(gpu):
  model = _model(F32, layers=1)
  ids, lens = torch.zeros((2, 4), dtype=torch.int64).cuda(), torch.tensor([4, 2]).cuda()
  timed = model.new_cache(2, 32, timestamps=True)
  with pytest.raises(ValueError, match="timestamps"):
    model.prefill(ids, timed, seq_lens=lens, timestamps=torch.zeros((2, 9), dtype=torch.int64).cuda(), ts_bias=torch.zeros(129).cuda())

  class Doubled(recml_amd.HSTUBlock):
    def forward(self, *args, **kw):
      return 2 * super().forward(*args, **kw)

  class Served(Doubled):
    def forward_cached(self, *args, **kw):
      return 2 * super().forward_cached(*args, **kw)

  block = model.decoder_blocks[0]
  block.__class__ = Doubled
  with pytest.raises(ValueError, match="forward_cached"):
    model.extend(ids, model.new_cache(2, 32))
  block.__class__ = Served
  assert model.extend(ids, model.new_cache(2, 32)).shape == (2, 4, 300)


@pytest.mark.parametrize("bits", [4, 8])
def test_two_blocks_with_times_event_by_event(gpu, bits):
  """An event's time bias reads the next event's time: in whatever calls events come in, what the second block keeps of them is the same,
  but for codes next to a border; and the last event's output is near the full call's."""
  model = _model(F32)
  B, L, n0 = 3, 40, 5
  ids = torch.randint(1, 300, (B, L), generator=_gen(1)).cuda()
  ts = (1_600_000_000 + torch.exp(torch.rand((B, L), generator=_gen(2)) * 15).long().cumsum(1)).cuda()
  kw = dict(pos_bias=(torch.randn((2, 2 * L - 1), generator=_gen(3)) * 0.2).cuda(), ts_bias=torch.randn((2, 129), generator=_gen(4)).cuda())
  caches = [model.new_cache(B, L, bits=bits, page_size=32, timestamps=True) for _ in range(3)]
  for c in caches:
    model.prefill(ids[:, :n0], c, seq_lens=torch.full((B,), n0).cuda(), timestamps=ts[:, :n0], **kw)
  together = model.extend(ids[:, n0:], caches[0], timestamps=ts[:, n0:], **kw)
  for i in range(n0, L):
    one = model.extend(ids[:, i : i + 1], caches[1], timestamps=ts[:, i : i + 1], **kw)
  for i in range(n0, L, 7):
    new, when = ids[:, i : i + 7], ts[:, i : i + 7]
    m = new.shape[1]
    some = model.extend(new.reshape(-1), caches[2], offsets=m * torch.arange(B + 1).cuda(), max_new=m, timestamps=when.reshape(-1), **kw)
  # Sums in another order move a value by 1e-5 of itself at most (the tolerance of the tests of one block), codes are at least 2^-4 of it apart:
  # of the first block's 30 thousand values less than 2e-5 * 2^4 of each, 10 in all, change their code.  One that does moves what later events get there by less
  # than 2^-3 of one of its 64 * 32 terms, 1e-3 of the sum's norm with its neighbours' signs, and with it 2 * 1e-3 * 2^4 = 3 in 100 of the second block's
  # codes.  (Kept as if each event were the last: 19 in 100 of the codes of 4 bits, 48 of those of 8.)
  for c in caches[1:]:
    for share, mine, other in zip((0.001, 0.05), caches[0].layers, c.layers):
      for a, b in ((mine.k, other.k), (mine.v, other.v)):
        assert float((a != b).float().mean()) <= share * L / 64
  full = model(ids, seq_lens=torch.full((B,), L).cuda(), timestamps=ts, **kw)
  # keys and values each off by at most 2^-4 (2^-2) of themselves, in two blocks, each beside a residual that is not
  assert float((together - full[:, n0:]).norm() / full[:, n0:].norm()) <= 4 * (2.0**-2 if bits == 4 else 2.0**-4)
  for last in (one[:, -1], some.reshape(B, m, -1)[:, -1]):
    assert float((last - full[:, -1]).norm() / full[:, -1].norm()) <= 4 * (2.0**-2 if bits == 4 else 2.0**-4)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prefill_with_times_is_the_forward(gpu, dtype, bits):
  """Both tables, two blocks, histories of every length up to the cache's; what is kept does not come into it."""
  model = _model(dtype)
  B, L, long = 5, 50, 44
  ids = torch.randint(1, 300, (B, long), generator=_gen(1)).cuda()
  ts = (1_600_000_000 + torch.exp(torch.rand((B, long), generator=_gen(2)) * 15).long().cumsum(1)).cuda()
  lens = torch.tensor([44, 1, 0, 33, 2]).cuda()
  kw = dict(pos_bias=(torch.randn((2, 2 * L - 1), generator=_gen(3)) * 0.2).cuda(), ts_bias=torch.randn((2, 129), generator=_gen(4)).cuda())
  cache = model.new_cache(B, L, bits=bits, page_size=32, timestamps=True)
  out = model.prefill(ids, cache, seq_lens=lens, timestamps=ts, **kw)
  # the full call of the cache's length: its normaliser and its tables' extent
  pad = lambda x: torch.cat([x, torch.zeros((B, L - long), dtype=x.dtype, device=x.device)], 1)
  want = model(pad(ids), seq_lens=lens, jagged=True, timestamps=pad(ts), **kw)[:, :long]
  # two runs of the same steps, rounded in other places: 2^-8 a step in bf16, sums in other orders in fp32
  assert (out.double() - want.double()).norm() / want.double().norm() <= (1e-5 if dtype == F32 else 8 * 2.0**-8)
  valid = torch.arange(long).cuda()[None] < lens[:, None]
  assert not out[~valid].any() and torch.equal(cache.lengths, lens.int()) and torch.equal(cache.timestamps[:, :long][valid], ts[valid])
  assert torch.equal(cache.ids[:, :long][valid], ids[valid])


def test_the_gradient_of_the_head_against_differences(gpu):
  """Along the gradient itself the loss rises by its norm: an error of one in a hundred shows."""
  model = _model(F32, vocab=97)
  model.requires_grad_(True)
  ids = torch.randint(1, 97, (3, 12), generator=_gen(1)).cuda()
  lens = torch.tensor([12, 5, 1]).cuda()
  nxt = torch.where(torch.arange(12, device="cuda")[None] < (lens - 1)[:, None], ids.roll(-1, 1), -1)
  def loss():
    got = model.log_probs(ids, nxt, entropy=True, seq_lens=lens)
    return -(got.log_probs.double().sum() + 0.1 * got.entropy.double().sum()) / 15
  w = model.reverse_embedding
  g = torch.autograd.grad(loss(), w)[0]
  size = float(g.double().norm())
  d, h = g / g.norm(), 4e-3
  with torch.no_grad():
    before = model(ids, seq_lens=lens)
    ends = []
    for s in (h, -2 * h):
      w.add_(s * d)
      ends.append(float(loss()))
      after = model(ids, seq_lens=lens) if s > 0 else after
    w.add_(h * d)
  # A row's logits move by up to m for a step of 1 along d: third derivatives of ln sum exp stay below (2 m)^3 / 10 (a third central moment of
  # values in a span of 2 m), the entropy's, a product of it with log probabilities of up to 12, below ten times that, of which a tenth counts.
  m = ((after - before) / h).abs().amax(-1).double()
  smooth = h * h / 6 * float(((2 * m) ** 3).sum()) * 0.2 / 15
  # 15 log probabilities and 36 tenths of an entropy, each off by 89 steps of 2^-24 and four of its size (up to 12), twice over 2 h; weights that
  # moved by h d and were rounded to 2^-24 of about 0.1, 64 of them a logit with rows of norm 8
  rounding = (15 + 3.6) / 15 * ((89 + 4 * 12) * 2.0**-24 + 8 * 0.1 * 2.0**-24) / h
  tol = smooth + rounding + 1e-4 * size
  assert tol <= 0.02 * size, (smooth, rounding, size)
  assert abs((ends[0] - ends[1]) / (2 * h) - size) <= tol, (ends, size, tol)


def test_a_packed_step_with_times_in_a_graph(gpu):
  """Offsets, ids and times are copied in between replays: users with no, one or several new events, as the eager calls have them."""
  model = _model(BF16)
  pos, tab = (torch.randn((2, 127), generator=_gen(3)) * 0.2).cuda(), torch.randn((2, 129), generator=_gen(4)).cuda()
  kw = dict(pos_bias=pos, ts_bias=tab)
  T, B = 5, 4
  seq, when0 = torch.randint(1, 300, (B, 10), generator=_gen(1)).cuda(), 1_600_000_000 + torch.arange(10 * B).reshape(B, 10).cuda() * 977
  caches = [model.new_cache(B, 64, bits=8, page_size=32, timestamps=True) for _ in range(2)]
  for c in caches:
    model.prefill(seq, c, seq_lens=torch.tensor([10, 0, 3, 7]).cuda(), timestamps=when0, **kw)
  ids, when, offsets = torch.ones(T, dtype=torch.int64).cuda(), torch.full((T,), 1_700_000_000).cuda(), torch.tensor([0, 1, 2, 3, 5], dtype=torch.int32).cuda()
  def step(cache):
    return model.extend(ids, cache, offsets=offsets, max_new=3, timestamps=when, **kw)
  keep = caches[1].lengths.clone()
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    step(caches[1])
  torch.cuda.current_stream().wait_stream(s)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step(caches[1])
  caches[1].lengths.copy_(keep)
  # (what the warm-up wrote past the kept lengths is the past of nobody)
  for n, ends in enumerate(([0, 1, 2, 3, 5], [0, 0, 3, 3, 5], [0, 2, 2, 2, 2], [1, 2, 2, 4, 5], [0, 3, 4, 5, 5])):
    ids.copy_(torch.randint(1, 300, (T,), generator=_gen(20 + n)))
    when.copy_(1_700_000_000 + 100_000 * n + torch.arange(T) * 333)
    offsets.copy_(torch.tensor(ends))
    graph.replay()
    want = step(caches[0])
    torch.cuda.synchronize()
    rows = slice(ends[0], ends[-1])
    assert torch.equal(out[rows], want[rows]), n
    assert torch.equal(caches[0].lengths, caches[1].lengths)
    for b, m in enumerate(caches[0].lengths.tolist()):
      assert torch.equal(caches[0].ids[b, :m], caches[1].ids[b, :m]) and torch.equal(caches[0].timestamps[b, :m], caches[1].timestamps[b, :m])
