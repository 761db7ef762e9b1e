"""The model's serving path with a cache that rounds nothing, in 64 bits on the CPU: what is left is which rows run, over what, and
where they go.  The operators below it are stood in for by their definitions."""

import pytest
import torch

import recml_amd
from recml_amd import hstu_cache_ops, hstu_ops
from tests import serve_reference as R

L, H, D, VOCAB = 24, 2, 16, 40


class Pages:
  """Keys and values as they are, [pages, heads, page_size, head_dim]."""

  def __init__(self, pages, size, heads, dim):
    self.k, self.v = (torch.full((pages, heads, size, dim), 7.0, dtype=torch.float64) for _ in range(2))

  @classmethod
  def empty(cls, pages, page_size, heads, head_dim, *, bits=4, device=None):
    return cls(pages, page_size, heads, head_dim)

  def row(self, table, b, place):
    size = self.k.shape[2]
    page = int(table[b, place // size]) if 0 <= place < table.shape[1] * size else -1
    return (page, place % size) if 0 <= page < self.k.shape[0] else None


def _rows(B, x, offsets, max_new):
  """Each sequence's rows of x."""
  if offsets is None:
    return [(b, slice(None)) for b in range(B)]
  ends = offsets.tolist()
  return [(slice(ends[b], min(ends[b + 1], ends[b] + max_new)),) for b in range(B)]


def _write(pages, k, v, table, starts, *, offsets=None, max_new=None):
  for b, at in enumerate(_rows(table.shape[0], k, offsets, max_new)):
    for t in range(k[at].shape[0]):
      row = pages.row(table, b, int(starts[b]) + t)
      if row is not None:
        pages.k[row[0], :, row[1]], pages.v[row[0], :, row[1]] = k[at][t], v[at][t]


def _attend(q, pages, table, lengths, *, max_len, offsets=None, max_new=None, n=None, alpha=1.0, pos_bias=None, timestamps=None, ts_bias=None):
  out = torch.zeros_like(q)
  for b, at in enumerate(_rows(table.shape[0], q, offsets, max_new)):
    rows = [pages.row(table, b, j) for j in range(max_len)]
    held = torch.tensor([r is not None for r in rows])
    k, v = (torch.stack([torch.zeros(q.shape[-2:], dtype=q.dtype) if r is None else t[r[0], :, r[1]] for r in rows]) for t in (pages.k, pages.v))
    out[at] = R.attention(q[at], k, v, length=int(lengths[b]), max_len=max_len, held=held, n=n, alpha=alpha, pos_bias=pos_bias,
                          timestamps=None if timestamps is None else timestamps[b], ts_bias=ts_bias)[0]
  return out


def _attention(q, k, v, *, seq_lens=None, seq_offsets=None, max_len=None, timestamps=None, bias=None, batch=None, **kw):
  """hstu_attention, padded or packed."""
  assert bias is None
  out = torch.zeros_like(q)
  if seq_offsets is None:
    seqs, max_len = [(b, slice(0, int(n))) for b, n in enumerate(seq_lens)], q.shape[1]
  else:
    seqs = _rows(len(seq_offsets) - 1, q, seq_offsets, max_len)
  for at in seqs:
    m = q[at].shape[0]
    if m:
      ts = None if timestamps is None else timestamps[at]
      out[at] = R.attention(q[at], k[at], v[at], length=m, max_len=max_len, held=torch.ones(m, dtype=torch.bool), timestamps=ts, **kw)[0]
  return out


@pytest.fixture(autouse=True)
def exact(monkeypatch):
  monkeypatch.setattr(hstu_cache_ops, "KVPages", Pages)
  monkeypatch.setattr(hstu_cache_ops, "kv_write", _write)
  monkeypatch.setattr(hstu_cache_ops, "cached_attention", _attend)
  monkeypatch.setattr(hstu_ops, "hstu_attention", _attention)


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _model(layers):
  m = recml_amd.HSTU(vocab_size=VOCAB, max_positions=L, model_dim=D, num_heads=H, num_layers=layers, scale_by_sqrt_dim=True, dtype=torch.float64, seed=5)
  g = _gen(6)
  for p in m.parameters():
    p.data.add_(torch.randn(p.shape, generator=g, dtype=torch.float64) * 0.1)
  return m.eval()


def _data(B=3, seed=1):
  ids = torch.randint(0, VOCAB, (B, L), generator=_gen(seed))
  # (gaps from a second to months, so that the next event's time and an event's own lie in other buckets)
  ts = 1_600_000_000 + torch.exp(torch.rand((B, L), generator=_gen(seed + 1)) * 15).long().cumsum(1)
  return ids, ts, torch.randn((H, 2 * L - 1), generator=_gen(seed + 2)).double() * 0.3, torch.randn((H, 129), generator=_gen(seed + 3)).double()


def _full(model, ids, ts, lens, kw, timed):
  return model(ids, seq_lens=torch.tensor(lens), **(dict(timestamps=ts, **kw) if timed else dict(pos_bias=kw["pos_bias"])))


def _same(got, want):
  # sums of a few dozen terms of about 1 in 64 bits, through norms and three layers
  assert got.shape == want.shape and bool(((got - want).abs() <= 1e-10).all())


# how the events of three users come in: counts a call
DEALT = {"one by one": [(1, 1, 1)] * 9, "together": [(9, 9, 9)], "in twos and threes": [(2, 2, 2), (3, 3, 3), (1, 1, 1), (3, 3, 3)],
         "unevenly": [(2, 0, 1), (0, 0, 3), (1, 4, 0), (0, 1, 0), (3, 2, 1)]}


@pytest.mark.parametrize("timed", [False, True])
@pytest.mark.parametrize("layers", [1, 2, 3])
@pytest.mark.parametrize("how", DEALT)
def test_extend_is_the_forward(how, layers, timed):
  """Whatever calls a user's events come in by, every row is the full call's on the events so far."""
  model, (ids, ts, pos, tab) = _model(layers), _data()
  kw = dict(pos_bias=pos, ts_bias=tab)
  step = lambda t: dict(timestamps=t, **kw) if timed else dict(pos_bias=pos)
  padded, packed = (model.new_cache(3, L, page_size=4, timestamps=timed) for _ in range(2))
  lens = [5, 0, 9]
  for c in (padded, packed):
    out = model.prefill(ids[:, :9], c, seq_lens=torch.tensor(lens), **step(ts[:, :9]))
    full = _full(model, ids, ts, lens, kw, timed)
    for b in range(3):
      _same(out[b, : lens[b]], full[b, : lens[b]])
  for counts in DEALT[how]:
    new = [(b, lens[b] + t) for b in range(3) for t in range(counts[b])]
    pick = lambda x: torch.stack([x[b, i] for b, i in new])
    ends = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()])
    lens = [n + c for n, c in zip(lens, counts)]
    full = _full(model, ids, ts, lens, kw, timed)
    out = model.extend(pick(ids), packed, offsets=ends, max_new=max(counts), **step(pick(ts)))
    for row, (b, i) in zip(out, new):
      _same(row, full[b, i])
    assert packed.lengths.tolist() == lens
    if len(set(counts)) == 1:
      out = model.extend(pick(ids).reshape(3, -1), padded, **step(pick(ts).reshape(3, -1)))
      _same(out, torch.stack([full[b, i] for b, i in new]).reshape(out.shape))
      assert padded.lengths.tolist() == lens


@pytest.mark.parametrize("layers", [1, 2])
def test_what_a_step_leaves_alone(layers):
  """Users without new events keep every bit, the others all but their last event and what comes behind it; rows of nobody and past max_new
  join nothing."""
  model, (ids, ts, pos, tab) = _model(layers), _data()
  kw = dict(pos_bias=pos, ts_bias=tab)
  cache = model.new_cache(3, L, page_size=4, timestamps=True)
  lens = [5, 3, 8]
  model.prefill(ids[:, :9], cache, seq_lens=torch.tensor(lens), timestamps=ts[:, :9], **kw)
  before = [(p.k.clone(), p.v.clone()) for p in cache.layers]
  # user 0: rows 1 and 2; user 1: none; user 2: rows 3, 4, 5, of which the last is past max_new
  rows = torch.tensor([7, int(ids[0, 5]), int(ids[0, 6]), int(ids[2, 8]), int(ids[2, 9]), 8, 9])
  when = torch.stack([ts[0, 0], ts[0, 5], ts[0, 6], ts[2, 8], ts[2, 9], ts[2, 10], ts[2, 11]])
  out = model.extend(rows, cache, offsets=torch.tensor([1, 3, 3, 6]), max_new=2, timestamps=when, **kw)
  assert out.shape == (7, VOCAB) and cache.lengths.tolist() == [7, 3, 10]
  full = _full(model, ids, ts, [7, 3, 10], kw, True)
  _same(out[1:5], torch.stack([full[0, 5], full[0, 6], full[2, 8], full[2, 9]]))
  each = L // 4
  for p, olds in zip(cache.layers, before):
    for now, old in zip((p.k, p.v), olds):
      by_place = lambda t, b: t[b * each : (b + 1) * each].transpose(1, 2).reshape(L, H, -1)
      for b, n in enumerate(lens):
        assert torch.equal(by_place(now, b)[: n - 1], by_place(old, b)[: n - 1])
      assert torch.equal(by_place(now, 1), by_place(old, 1))
      for b, n in ((0, 7), (2, 10)):
        assert torch.equal(by_place(now, b)[n:], by_place(old, b)[n:])


def test_a_history_that_is_full():
  """Events past the cache's end are lost; the last one that is kept is the forward's, and stays so."""
  model, (ids, ts, pos, tab) = _model(2), _data()
  kw = dict(pos_bias=pos, ts_bias=tab)
  cache = model.new_cache(3, L, page_size=4, timestamps=True)
  lens = [L - 1, L, L - 3]
  model.prefill(ids, cache, seq_lens=torch.tensor(lens), timestamps=ts, **kw)
  more, late = torch.full((3, 2), 5), ts[:, -1:] + torch.tensor([[10, 20]])
  new = torch.stack([torch.stack([ids[0, L - 1], more[0, 0]]), more[1], ids[2, L - 3 : L - 1]])
  when = torch.stack([torch.stack([ts[0, L - 1], late[0, 0]]), late[1], ts[2, L - 3 : L - 1]])
  whole = [(p.k[L // 4 : L // 2].clone(), p.v[L // 4 : L // 2].clone()) for p in cache.layers]
  out = model.extend(new, cache, timestamps=when, **kw)
  full = _full(model, ids, ts, [L, L, L - 1], kw, True)
  _same(out[0, 0], full[0, L - 1])
  _same(out[2], full[2, L - 3 : L - 1])
  for p, old in zip(cache.layers, whole):
    assert torch.equal(p.k[L // 4 : L // 2], old[0]) and torch.equal(p.v[L // 4 : L // 2], old[1])
  kept = [(p.k[: L // 4].clone(), p.v[: L // 4].clone()) for p in cache.layers]
  out = model.extend(torch.stack([more[0, :1], more[1, :1], ids[2, L - 1 :]]), cache, timestamps=torch.stack([late[0, 1:], late[1, 1:], ts[2, L - 1 :]]), **kw)
  _same(out[2, 0], _full(model, ids, ts, [L, L, L], kw, True)[2, L - 1])
  for p, old in zip(cache.layers, kept):
    assert torch.equal(p.k[: L // 4], old[0]) and torch.equal(p.v[: L // 4], old[1])


def test_rewound_and_begun_again():
  """Lengths set back by the caller, and users reset: what comes next follows what is kept."""
  model, (ids, ts, pos, tab) = _model(3), _data()
  kw = dict(pos_bias=pos, ts_bias=tab)
  other, when, _, _ = _data(seed=31)
  when = torch.maximum(when, ts)
  cache = model.new_cache(3, L, page_size=4, timestamps=True)
  model.prefill(ids[:, :9], cache, seq_lens=torch.tensor([9, 4, 6]), timestamps=ts[:, :9], **kw)
  mixed, at = ids.clone(), ts.clone()
  for b, n in ((0, 9), (1, 4), (2, 6)):
    model.extend(other[b, n : n + 3], cache, offsets=torch.tensor([0] * (b + 1) + [3] * (3 - b)), max_new=3, timestamps=when[b, n : n + 3], **kw)
    mixed[b, n : n + 1], at[b, n : n + 1] = other[b, n : n + 1], when[b, n : n + 1]
  cache.lengths.copy_(torch.tensor([10, 5, 7]))
  cache.reset(torch.tensor([1]))
  mixed[1], at[1] = ids[1], ts[1]
  lens, at = [10, 0, 7], at.cummax(1).values
  pick = lambda x: torch.stack([x[b, n : n + 2] for b, n in enumerate(lens)])
  out = model.extend(pick(mixed), cache, timestamps=pick(at), **kw)
  full = _full(model, mixed, at, [n + 2 for n in lens], kw, True)
  _same(out, torch.stack([full[b, n : n + 2] for b, n in enumerate(lens)]))


@pytest.mark.parametrize("everywhere", [False, True])
def test_hooks_run(everywhere):
  """Hooks on the blocks, or on all modules, do in serving what they do in the model's call."""
  model, (ids, ts, pos, tab) = _model(2), _data()
  kw = dict(pos_bias=pos, ts_bias=tab)
  seen = []
  def before(module, args):
    if isinstance(module, recml_amd.HSTUBlock):
      return (args[0] * 1.5,)
  def after(module, args, out):
    if isinstance(module, recml_amd.HSTUBlock):
      seen.append(tuple(out.shape))
      return out - 0.25
  m = torch.nn.modules.module
  if everywhere:
    handles = [m.register_module_forward_pre_hook(before), m.register_module_forward_hook(after)]
  else:
    handles = [model.decoder_blocks[0].register_forward_pre_hook(before), model.decoder_blocks[1].register_forward_hook(after)]
  try:
    cache = model.new_cache(3, L, page_size=4, timestamps=True)
    out = model.prefill(ids[:, :9], cache, seq_lens=torch.tensor([9, 0, 4]), timestamps=ts[:, :9], **kw)
    assert seen == [(13, D)] * len(seen) and len(seen) == (2 if everywhere else 1)
    full = _full(model, ids, ts, [9, 0, 4], kw, True)
    _same(out[0], full[0, :9])
    new = lambda x: torch.stack([x[0, 9:11], x[1, 0:2], x[2, 4:6]])
    out = model.extend(new(ids), cache, timestamps=new(ts), **kw)
    _same(out, new(_full(model, ids, ts, [11, 2, 6], kw, True)))
  finally:
    for h in handles:
      h.remove()
  plain = model.new_cache(3, L, page_size=4, timestamps=True)
  assert not torch.equal(model.extend(ids[:, :1], plain, timestamps=ts[:, :1], **kw), out[:, :1])


def test_pruned_weights_are_served():
  """Pruning works its weights out in a hook ahead of each call."""
  from torch.nn.utils import prune
  model, (ids, _, pos, _) = _model(2), _data()
  prune.l1_unstructured(model.decoder_blocks[0], "v_kernel", amount=0.5)
  with torch.no_grad():
    model.decoder_blocks[0].v_kernel_orig.mul_(1.25)
  cache = model.new_cache(3, L, page_size=4)
  out = model.extend(ids[:, :4], cache, pos_bias=pos)
  _same(out, _full(model, ids, None, [4, 4, 4], dict(pos_bias=pos), False)[:, :4])


def test_hooks_around_another_forward_are_refused():
  """A subclass that serves through a forward_cached of its own: the hooks' place is around its forward, which is not run."""
  class Served(recml_amd.HSTUBlock):
    def forward(self, *args, **kw):
      return 2 * super().forward(*args, **kw)

    def forward_cached(self, *args, **kw):
      return 2 * super().forward_cached(*args, **kw)

  model, (ids, _, _, _) = _model(2), _data()
  model.decoder_blocks[1].__class__ = Served
  _same(model.extend(ids[:, :4], model.new_cache(3, L, page_size=4)), _full(model, ids, None, [4, 4, 4], dict(pos_bias=None), False)[:, :4])
  handle = model.decoder_blocks[1].register_forward_hook(lambda *a: None)
  with pytest.raises(ValueError, match="hooks"):
    model.extend(ids[:, :4], model.new_cache(3, L, page_size=4))
  handle.remove()
  model.decoder_blocks[0].register_forward_hook(lambda *a: None)
  assert model.extend(ids[:, :4], model.new_cache(3, L, page_size=4)).shape == (3, 4, VOCAB)
