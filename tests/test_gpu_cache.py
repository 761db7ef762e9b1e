"""The cache of keys and values in 4 and 8 bits and the attention over it, against their definitions in 64 bits."""

import math

import pytest
import torch

import recml_amd
from tests import serve_reference as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _table(lengths, page, spare, seed, most=None):
  """Pages in no order; entries past a sequence's end name none."""
  held = [-(-n // page) for n in lengths]
  most = max(held) if most is None else most
  free = torch.randperm(sum(held) + spare, generator=_gen(seed)).tolist()
  t = torch.full((len(lengths), most), -1, dtype=torch.int32)
  for b, n in enumerate(held):
    for i in range(n):
      t[b, i] = free.pop()
  return t, sum(held) + spare


def _pages(pages, page, H, d, bits, garbage=True):
  got = recml_amd.KVPages.empty(pages, page, H, d, bits=bits, device="cuda:0")
  if garbage:                # what earlier histories left there, codes and exponents that are no numbers among it
    for t in (got.k, got.v, got.k_scales, got.v_scales):
      t.copy_(torch.randint(0, 256, t.shape, generator=_gen(5), dtype=torch.uint8))
      t.view(-1)[::7] = 255
  return got


def _at(table, page, b, place):
  i = place // page
  return (int(table[b, i]), place % page) if 0 <= i < table.shape[1] else (-1, 0)


def _rows_of(shape, dtype, seed, scale=0.3):
  x = torch.randn(shape, generator=_gen(seed)) * scale
  # blocks at many powers, a block of zeros, values on the borders between codes
  x = x * torch.exp2(torch.randint(-12, 13, shape[:-1] + (1,), generator=_gen(seed + 1)).float())
  flat = x.view(-1, shape[-1])
  flat[0] = 0
  if len(flat) > 2:
    flat[2, : min(16, shape[-1])] = torch.tensor([7, 6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.25, -5, 4, 464, 456, 448, -7])[: shape[-1]]
  if len(flat) > 3:
    flat[3] = 0
    flat[3, :8] = torch.tensor([7.03125, 6, 5, 3.5, 2.5, 1.75, 0.25, -1.25])
  if len(flat) > 4:
    flat[4] = flat[4] * 0 + 2.0**-126
  if len(flat) > 5:
    flat[5, 0] = 3e38
  return x.to(dtype)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", recml_amd.hstu_cache_ops.HEAD_DIMS)
def test_rows_are_stored_as_defined(gpu, bits, dtype, d):
  H, page, starts, n = 3, 32, [0, 5, 31, 63], 37
  table, pages = _table([s + n for s in starts], page, 3, 1)
  got = _pages(pages, page, H, d, bits)
  before = [t.clone() for t in (got.k, got.k_scales, got.v, got.v_scales)]
  k, v = (_rows_of((4, n, H, d), dtype, s) for s in (1, 2))
  recml_amd.kv_write(got, k.cuda(), v.cuda(), table.cuda(), torch.tensor(starts).cuda())
  torch.cuda.synchronize()
  touched = torch.zeros((pages, page), dtype=torch.bool)
  for x, codes, scales in ((k, got.k, got.k_scales), (v, got.v, got.v_scales)):
    held = R.values(codes.cpu(), scales.cpu(), bits, d)
    want = R.stored(x, bits)
    for b, s in enumerate(starts):
      for t in range(n):
        p, slot = _at(table, page, b, s + t)
        touched[p, slot] = True
        assert torch.equal(held[p, :, slot], want[b, t]), (b, t)
  # every other row is as it was
  for t, was in zip((got.k, got.v), before[0::2]):
    assert torch.equal(t.cpu()[~touched[:, None, :].expand(pages, H, page)], was.cpu()[~touched[:, None, :].expand(pages, H, page)])
  for t, was in zip((got.k_scales, got.v_scales), before[1::2]):
    at = ~touched[:, None, None, :].expand(t.shape)
    assert torch.equal(t.cpu()[at], was.cpu()[at])
  for out in (BF16, F32):
    rk, rv = recml_amd.kv_read(got, table.cuda(), torch.tensor(starts).cuda(), count=n, dtype=out)
    for r, x in ((rk, k), (rv, v)):
      want = R.stored(x, bits)
      assert r.dtype == out and torch.equal(r.cpu().double(), want.to(out).double())


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_that_are_not_finite_read_back_as_nan(gpu, bits):
  H, d, page = 2, 96, 64
  x = torch.randn((1, 6, H, d), generator=_gen(3))
  x[0, 1, 0, 5], x[0, 2, 1, 95], x[0, 4, 0, 40] = math.inf, -math.inf, math.nan
  got = _pages(2, page, H, d, bits)
  table = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
  recml_amd.kv_write(got, x.cuda(), x.cuda(), table, torch.tensor([60]).cuda())
  for r in recml_amd.kv_read(got, table, torch.tensor([60]).cuda(), count=6, dtype=F32):
    r, want = r.cpu(), R.stored(x, bits)
    assert torch.equal(torch.isnan(r), torch.isnan(want)) and torch.isnan(r[0, 1, 0]).all() and not torch.isnan(r[0, 1, 1]).any()
    assert torch.equal(torch.nan_to_num(r.double()), torch.nan_to_num(want))


@pytest.mark.parametrize("bits,d,page", [(4, 128, 64), (8, 48, 96), (4, 16, 32)])
def test_packed_rows_and_places_without_a_page(gpu, bits, d, page):
  H, counts, starts = 2, [0, 3, 70, 1, 33], [4, -2, 60, 5 * page - 1, 0]
  most = 3
  table, pages = _table([2 * page] * 5, page, 1, 7, most)
  table[4, 0] = pages                      # one past the last page
  offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int64)
  T = int(offsets[-1]) + 2                 # two rows behind the last sequence
  got = _pages(pages, page, H, d, bits)
  before = [t.cpu().clone() for t in (got.k, got.v)]
  k, v = (_rows_of((T, H, d), BF16, s) for s in (11, 12))
  how = dict(offsets=offsets.cuda(), max_new=max(counts))
  recml_amd.kv_write(got, k.cuda(), v.cuda(), table.cuda(), torch.tensor(starts).cuda(), **how)
  rk, rv = recml_amd.kv_read(got, table.cuda(), torch.tensor(starts).cuda(), total=T, **how)
  touched = torch.zeros((pages, page), dtype=torch.bool)
  for x, r, codes, was in ((k, rk, got.k, before[0]), (v, rv, got.v, before[1])):
    want = R.stored(x, bits)
    for b in range(5):
      for t in range(counts[b]):
        p, slot = _at(table, page, b, starts[b] + t)
        row = int(offsets[b]) + t
        if 0 <= p < pages and starts[b] + t >= 0:
          touched[p, slot] = True
          assert torch.equal(r[row].cpu().double(), want[row]), (b, t)
        else:
          assert not r[row].any()
    at = ~touched[:, None, :].expand(pages, H, page)
    assert torch.equal(codes.cpu()[at], was[at])


def _case(*, B, H, d, bits, page, lengths, counts, max_len, dtype, packed, seed, pos=None, ts=None, alpha=1.0, n=None, most=None, strided=False,
          nb=128, bucket_size=0.301):
  """Caches filled by kv_write with values of kept rows on both sides of zero; returns the call and the reference's rows."""
  table, pages = _table(lengths, page, 2, seed, most)
  got = _pages(pages, page, H, d, bits)
  places = table.shape[1] * page
  k, v = (torch.randn((B, max(lengths) if lengths else 1, H, d), generator=_gen(seed + i)) * 0.4 for i in (1, 2))
  lens = torch.tensor(lengths, dtype=torch.int32)
  offs = torch.tensor([0, *lens.cumsum(0).tolist()], dtype=torch.int32)
  flat = lambda x: torch.cat([x[b, : lengths[b]] for b in range(B)])
  recml_amd.kv_write(got, flat(k).cuda(), flat(v).cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32).cuda(), offsets=offs.cuda(),
                     max_new=max(lengths))
  m = max(counts)
  q = (torch.randn((B, m, H, d), generator=_gen(seed + 3)) * 0.5).to(dtype)
  kw = dict(max_len=max_len, alpha=alpha, n=n)
  if pos:
    kw["pos_bias"] = torch.randn((H if pos == "heads" else 1, 2 * max_len - 1), generator=_gen(seed + 4)) * 0.5
  if ts:
    gaps = torch.randint(0, 3 * 10 ** 4, (B, max_len), generator=_gen(seed + 5)) ** 2 // 100
    kw["timestamps"] = 1_600_000_000 + gaps.cumsum(1)
    kw["ts_bias"] = torch.randn((H if ts == "heads" else 1, nb + 1), generator=_gen(seed + 6)) * 0.5
    kw["ts_bucket_size"] = bucket_size
  call = {name: x.cuda() if isinstance(x, torch.Tensor) else x for name, x in kw.items()}
  if packed:
    qo = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
    rows = torch.cat([q[b, : counts[b]] for b in range(B)] + [torch.full((2, H, d), 7.0, dtype=dtype)])
    call.update(offsets=qo.cuda(), max_new=m)
  else:
    assert len(set(counts)) == 1
    rows = q
  rows = rows.cuda()
  if strided:                # a slice of a fused projection
    wide = torch.zeros((*rows.shape[:-2], 3, *rows.shape[-2:]), dtype=dtype, device="cuda")
    wide[..., 1, :, :] = rows
    rows = wide[..., 1, :, :]
  held_k, held_v = (R.values(c.cpu(), s.cpu(), bits, d) for c, s in ((got.k, got.k_scales), (got.v, got.v_scales)))
  want = []
  for b in range(B):
    at = [_at(table, page, b, j) for j in range(places)]
    held = torch.tensor([0 <= p < pages for p, _ in at], dtype=torch.bool)
    kk, vv = (torch.stack([x[p, :, s] if 0 <= p < pages else torch.zeros((H, d), dtype=torch.float64) for p, s in at]) for x in (held_k, held_v))
    ref = dict(kw)
    if ts:
      ref["timestamps"] = kw["timestamps"][b]
    want.append(R.attention(q[b, : counts[b]], kk, vv, length=lengths[b], held=held, **ref))
  return got, rows, table.cuda(), lens.cuda(), call, want, counts


def _compare(out, want, counts, packed, lengths, dtype):
  row = 0
  for b, (ref, off, weights) in enumerate(want):
    mine = out[row : row + counts[b]] if packed else out[b, : counts[b]]
    row += counts[b]
    mine = mine.cpu().double()
    tol = R.attention_tolerance(ref, off, weights, lengths[b], dtype)
    assert torch.equal(torch.isnan(mine), torch.isnan(ref)), b
    bad = ((mine - ref).abs() > tol).nan_to_num(0).bool() & ~torch.isnan(ref)
    assert not bad.any(), (b, float((mine - ref).abs().nan_to_num(0).max()), float(tol.max()))


SHAPES = [
    # B, H, d, bits, page, lengths, counts, max_len
    (1, 1, 128, 4, 64, [1], [1], 1),
    (2, 2, 128, 4, 64, [65, 64], [1, 1], 70),
    (3, 8, 128, 4, 64, [1000, 33, 517], [1, 1, 1], 1024),
    (2, 2, 128, 8, 32, [300, 31], [1, 1], 301),
    (3, 3, 64, 8, 96, [200, 5, 97], [24, 3, 17], 250),
    (2, 2, 64, 4, 64, [130, 129], [40, 40], 131),
    (2, 1, 32, 4, 32, [100, 7], [5, 7], 100),
    (2, 4, 16, 8, 32, [50, 9], [2, 2], 50),
    (1, 2, 8, 4, 32, [70], [3], 99),
    (1, 2, 24, 8, 64, [70], [70], 70),
    (2, 2, 48, 4, 64, [90, 64], [1, 33], 90),
    (1, 3, 96, 8, 64, [400], [66], 400),
    (1, 1, 192, 4, 64, [210], [20], 210),
    (2, 2, 256, 8, 64, [129, 300], [1, 2], 300),
    (1, 2, 256, 4, 32, [90], [40], 90),
    (1, 2, 128, 4, 128, [2500], [129], 2500),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])) + "-" + str(max(s[5])))
def test_attention_over_the_cache(gpu, shape, dtype):
  B, H, d, bits, page, lengths, counts, max_len = shape
  packed = len(set(counts)) > 1
  pos, ts = (("heads", None), ("heads", "one"), (None, None), ("one", "heads"))[(B + d // 8 + bits) % 4]
  got, rows, table, lens, call, want, counts = _case(B=B, H=H, d=d, bits=bits, page=page, lengths=lengths, counts=counts, max_len=max_len,
                                                     dtype=dtype, packed=packed, seed=d + bits, pos=pos, ts=ts, alpha=0.7, strided=bool(H % 2))
  out = recml_amd.cached_attention(rows, got, table, lens, **call)
  assert out.dtype == dtype and out.shape == rows.shape
  _compare(out, want, counts, packed, lengths, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_attend_to_nothing(gpu, dtype):
  """Lengths of zero, rows at places below 0 and at places past the table or max_len, pages that nobody has."""
  lengths, counts = [3, 40, 150, 1], [5, 5, 5, 5]
  table, pages = _table([3, 40, 128, 1], 32, 2, 3, 4)
  H, d, L = 2, 64, 140
  got = _pages(pages, 32, H, d, 4)
  k = torch.randn((4, 128, H, d), generator=_gen(1)) * 0.4
  zero = torch.zeros(4, dtype=torch.int32).cuda()
  recml_amd.kv_write(got, k.cuda(), k.flip(0).cuda(), table.cuda(), zero)
  table[1, 0] = -1                                         # the second sequence's oldest page is gone
  table[0, 0] = pages + 3
  q = (torch.randn((4, 5, H, d), generator=_gen(2)) * 0.5).to(dtype)
  lens = torch.tensor([3, 40, 150, 0], dtype=torch.int32)
  out = recml_amd.cached_attention(q.cuda(), got, table.cuda(), lens.cuda(), max_len=L)
  held_k, held_v = (R.values(c.cpu(), s.cpu(), 4, d) for c, s in ((got.k, got.k_scales), (got.v, got.v_scales)))
  for b in range(4):
    at = [_at(table, 32, b, j) for j in range(128)]
    held = torch.tensor([0 <= p < pages for p, _ in at], dtype=torch.bool)
    kk, vv = (torch.stack([x[p, :, s] if 0 <= p < pages else torch.zeros((H, d), dtype=torch.float64) for p, s in at]) for x in (held_k, held_v))
    ref, off, weights = R.attention(q[b], kk, vv, length=int(lens[b]), held=held, max_len=L)
    tol = R.attention_tolerance(ref, off, weights, 128, dtype)
    mine = out[b].cpu().double()
    assert ((mine - ref).abs() <= tol).all(), b
    if b in (0, 2, 3):
      assert not mine.any()                                # no page, places past the table's 128, no events at all
  assert out[1].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_kept_rows_that_are_no_numbers(gpu, bits, dtype):
  """A key or value that is not finite is NaN for the queries that attend to it and nothing for the others."""
  H, d, page, L = 2, 96, 32, 70
  table, pages = _table([L], page, 1, 2)
  got = _pages(pages, page, H, d, bits)
  k, v = (torch.randn((1, L, H, d), generator=_gen(s)) * 0.4 for s in (1, 2))
  k[0, 66, 0, 3], v[0, 68, 1, 90] = math.inf, math.nan
  recml_amd.kv_write(got, k.cuda(), v.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32).cuda())
  q = (torch.randn((1, 6, H, d), generator=_gen(3)) * 0.5).to(dtype)
  out = recml_amd.cached_attention(q.cuda(), got, table.cuda(), torch.tensor([L]).cuda(), max_len=L).cpu()
  nan = torch.isnan(out[0])
  for t in range(6):
    assert nan[t, 0].all() == (t >= 2) and nan[t, 0].any() == (t >= 2), t
    assert nan[t, 1].all() == (t >= 4) and nan[t, 1].any() == (t >= 4), t


def test_timestamps_on_the_borders_of_buckets(gpu):
  """Every bucket's first difference and the one before it, and differences of either sign."""
  size = 0.301
  edges = sorted({max(1, math.ceil(math.exp(b * float(torch.tensor(size))) + o)) for b in range(70) for o in (-2, -1, 0, 1)})
  edges = [e for e in edges if e < 10**9] + [10**9, 10**9 + 5, 10**12, 0]
  L = len(edges) + 1
  ts = torch.tensor([[10**13 - e for e in edges] + [10**13]])
  ts[0, ::3] = 2 * 10**13 - ts[0, ::3]
  ts[0, -1] = 10**13
  H, d, page = 1, 32, 32
  table, pages = _table([L], page, 0, 2)
  got = recml_amd.KVPages.empty(pages, page, H, d, bits=8, device="cuda:0")
  k, v = torch.zeros((1, L, H, d)), torch.zeros((1, L, H, d))
  tab = torch.arange(129).float() + 20.0                    # (silu(x) = x here, to 2e-9)
  for first in range(0, L, d):                              # each key's weight on a dim of its own
    v.zero_()
    for c in range(min(d, L - first)):
      v[0, first + c, 0, c] = 1.0
    recml_amd.kv_write(got, k.cuda(), v.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32).cuda())
    q = torch.zeros((1, 1, H, d))
    out = recml_amd.cached_attention(q.cuda(), got, table.cuda(), torch.tensor([L]).cuda(), max_len=L, n=1.0, timestamps=ts.cuda(),
                                     ts_bias=tab.cuda(), ts_bucket_size=size).cpu()[0, 0, 0]
    want = tab[R.bucket(ts[0, -1] - ts[0, first : first + d]).clamp(max=128)]
    assert torch.allclose(out[: len(want)], want, rtol=1e-6, atol=0), first


@pytest.mark.parametrize("nb,size", [(0, 0.301), (5, 0.301), (128, 0.05), (128, 3.0)])
def test_other_buckets(gpu, nb, size):
  got, rows, table, lens, call, want, counts = _case(B=2, H=2, d=32, bits=8, page=32, lengths=[90, 40], counts=[2, 2], max_len=90, dtype=F32,
                                                     packed=False, seed=4, ts="heads", nb=nb, bucket_size=size)
  _compare(recml_amd.cached_attention(rows, got, table, lens, **call), want, counts, False, [90, 40], F32)


def test_rows_of_no_sequence_are_left(gpu):
  got, rows, table, lens, call, want, counts = _case(B=2, H=2, d=64, bits=4, page=64, lengths=[700, 20], counts=[3, 1], max_len=700, dtype=BF16,
                                                     packed=True, seed=8)
  out = torch.full_like(rows, 3.0)
  assert recml_amd.cached_attention(rows, got, table, lens, out=out, **call) is out
  assert (out[4:] == 3.0).all()
  _compare(out, want, counts, True, [700, 20], BF16)


def test_the_same_bits_every_time_and_in_a_graph(gpu):
  """Replays of two captured calls and eager ones between them."""
  cases = [_case(B=3, H=4, d=128, bits=b, page=64, lengths=[900, 70, 1500], counts=[1, 1, 1], max_len=2048, dtype=BF16, packed=False, seed=b,
                 pos="heads", ts="heads") for b in (4, 8)]
  eager = [recml_amd.cached_attention(c[1], c[0], c[2], c[3], **c[4]) for c in cases]
  outs, graphs = [], []
  for c in cases:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(recml_amd.cached_attention(c[1], c[0], c[2], c[3], **c[4]))
    graphs.append(g)
  for _ in range(3):
    for g, o in zip(graphs, outs):
      o.zero_()
      g.replay()
    again = [recml_amd.cached_attention(c[1], c[0], c[2], c[3], **c[4]) for c in cases]
    torch.cuda.synchronize()
    for e, o, a in zip(eager, outs, again):
      assert torch.equal(e, o) and torch.equal(e, a)


def test_another_stream(gpu):
  c = _case(B=2, H=2, d=64, bits=4, page=64, lengths=[300, 20], counts=[1, 1], max_len=300, dtype=BF16, packed=False, seed=8)
  want = recml_amd.cached_attention(c[1], c[0], c[2], c[3], **c[4])
  torch.cuda.synchronize()
  s = torch.cuda.Stream()
  with torch.cuda.stream(s):
    got = recml_amd.cached_attention(c[1], c[0], c[2], c[3], **c[4])
  s.synchronize()
  assert torch.equal(got, want)


def test_a_step_as_it_is_served(gpu):
  """Events one by one: written, attended from, and the whole sequence again by hstu_attention over what the cache stands for."""
  B, H, d, page, L, first = 2, 2, 64, 32, 80, [37, 60]
  table, pages = _table([L, L], page, 0, 5)
  got = recml_amd.KVPages.empty(pages, page, H, d, bits=8, device="cuda:0")
  q, k, v = ((torch.randn((B, L, H, d), generator=_gen(s)) * 0.4).to(BF16).cuda() for s in (1, 2, 3))
  pos = (torch.randn((H, 2 * L - 1), generator=_gen(4)) * 0.3).cuda()
  ts = (1_600_000_000 + torch.randint(1, 10**5, (B, L), generator=_gen(5)).cumsum(1)).cuda()
  tab = (torch.randn((H, 129), generator=_gen(6)) * 0.3).cuda()
  table, lens = table.cuda(), torch.tensor(first, dtype=torch.int32).cuda()
  offs = torch.tensor([0, *torch.tensor(first).cumsum(0).tolist()], dtype=torch.int32).cuda()
  recml_amd.kv_write(got, *(torch.cat([x[b, : first[b]] for b in range(B)]) for x in (k, v)), table, torch.zeros_like(lens), offsets=offs, max_new=max(first))
  for step in range(8):
    new = [torch.stack([x[b, first[b] + step] for b in range(B)])[:, None] for x in (q, k, v)]
    recml_amd.kv_write(got, new[1], new[2], table, lens)
    lens = lens + 1
    out = recml_amd.cached_attention(new[0], got, table, lens, max_len=L, pos_bias=pos, timestamps=ts, ts_bias=tab)
    kk, vv = recml_amd.kv_read(got, table, torch.zeros_like(lens), count=L)
    whole = recml_amd.hstu_attention(q, kk, vv, seq_lens=lens, pos_bias=pos, timestamps=torch.where(
        torch.arange(L, device="cuda")[None] < lens[:, None], ts, ts.gather(1, (lens[:, None] - 1).long())), ts_bias=tab)
    want = torch.stack([whole[b, first[b] + step] for b in range(B)])[:, None]
    # two bf16 results of the same sums, each off by 2^-8 of its weights' magnitude and of itself
    size = (vv.abs().float().amax() * L * 2.0) / L
    assert (out.float() - want.float()).abs().max() <= 2 * 2.0**-8 * size


@pytest.mark.parametrize("packed", [False, True])
def test_the_python_way(gpu, monkeypatch, packed):
  """What the native host side declines goes through the Python one: the same kernels, the same bits."""
  from recml_amd import _native
  counts = [3, 1] if packed else [2, 2]
  got, rows, table, lens, call, want, counts = _case(B=2, H=2, d=64, bits=4, page=64, lengths=[700, 20], counts=counts, max_len=700, dtype=BF16,
                                                     packed=packed, seed=8, pos="heads", ts="one")
  how = dict(offsets=call["offsets"], max_new=call["max_new"]) if packed else {}
  read = dict(how, total=rows.shape[0]) if packed else dict(count=2)
  def step():
    recml_amd.kv_write(got, rows, rows * 0.5, table, lens - 3, **how)
    return [recml_amd.cached_attention(rows, got, table, lens, **call), *recml_amd.kv_read(got, table, lens - 3, **read)]
  native = step()
  for t in (got.k, got.v):
    t[int(table[1, 0]), :, 17:18] = 0                      # (a row that the next step writes again)
  for name in ("kv_write", "kv_read", "cached_attention"):
    monkeypatch.setattr(_native, name, lambda *a: None)
  T = sum(counts)
  for a, b in zip(native, step()):
    assert torch.equal(a[:T], b[:T])


def test_python_conversions_and_refusals(gpu):
  """64-bit lengths, misaligned and strided rows, tables of other types; and what is refused."""
  got, rows, table, lens, call, want, counts = _case(B=2, H=2, d=64, bits=8, page=64, lengths=[130, 20], counts=[2, 2], max_len=130, dtype=BF16,
                                                     packed=False, seed=9, pos="heads", ts="one")
  native = recml_amd.cached_attention(rows, got, table, lens, **call)
  odd = torch.zeros(rows.numel() + 1, dtype=BF16, device="cuda")[1:].view(rows.shape)
  odd.copy_(rows)
  other = dict(call, pos_bias=call["pos_bias"].double(), ts_bias=call["ts_bias"].double(), timestamps=call["timestamps"].t().contiguous().t())
  assert torch.equal(native, recml_amd.cached_attention(odd, got, table.long(), lens.long(), **other))
  assert torch.equal(native, recml_amd.cached_attention(rows.transpose(2, 3).contiguous().transpose(2, 3), got, table, lens, **call))
  bad = [dict(q=rows[:1]), dict(q=rows[..., :32]), dict(q=rows.half()), dict(lengths=lens[:1]), dict(lengths=lens.float()), dict(max_len=0), dict(n=0.0), dict(n=-1),
         dict(pos_bias=call["pos_bias"][:, 1:]), dict(timestamps=None), dict(timestamps=call["timestamps"][:, 1:]), dict(ts_bias=torch.zeros(130, device="cuda")),
         dict(out=rows.float()), dict(out=odd), dict(page_table=table[0]), dict(page_table=table.float()), dict(max_new=7), dict(lengths=lens.cpu()),
         dict(offsets=torch.tensor([0, 2, 4]).cuda())]
  for change in bad:
    args = dict(call, q=rows, page_table=table, lengths=lens)
    args.update(change)
    with pytest.raises(ValueError):
      recml_amd.cached_attention(args.pop("q"), got, args.pop("page_table"), args.pop("lengths"), **args)
  leaf = rows.clone().requires_grad_(True)
  with pytest.raises(ValueError, match="no gradient"):
    recml_amd.cached_attention(leaf, got, table, lens, **call)
  with pytest.raises(ValueError, match="no gradient"):
    recml_amd.kv_write(got, leaf, rows, table, lens)
  with torch.no_grad():
    assert torch.equal(native, recml_amd.cached_attention(leaf, got, table, lens, **call))
  for how in (dict(), dict(count=-1), dict(count=2, total=3), dict(offsets=torch.tensor([0, 1, 2]).cuda()), dict(count=1, dtype=torch.float16)):
    with pytest.raises(ValueError):
      recml_amd.kv_read(got, table, lens, **how)
  with pytest.raises(AttributeError):
    got.k = got.v
  for parts in ((got.k[:, :, :31], got.k_scales, got.v, got.v_scales), (got.k, got.k_scales[..., 1:], got.v, got.v_scales), (got.k.float(), got.k_scales, got.v, got.v_scales),
                (got.k, got.k_scales, got.v[:1], got.v_scales)):
    with pytest.raises(ValueError):
      recml_amd.KVPages(*parts, head_dim=64)


def test_pages_past_four_gigabytes(gpu):
  """Codes at offsets that 32 bits do not hold."""
  H, d, page, pages, n = 2, 256, 128, 70_000, 300                 # (64 KB a page: 4.6 GB of codes, keys and values each)
  got = recml_amd.KVPages.empty(pages, page, H, d, bits=8, device="cuda:0")
  assert got.k.numel() > 2**32
  table = torch.tensor([[69_999, 3, 69_998]], dtype=torch.int32)
  k, v = (torch.randn((1, n, H, d), generator=_gen(s)) * 0.4 for s in (1, 2))
  q = torch.randn((1, 2, H, d), generator=_gen(3)) * 0.4
  zero = torch.zeros(1, dtype=torch.int32).cuda()
  recml_amd.kv_write(got, k.cuda(), v.cuda(), table.cuda(), zero)
  for r, x in zip(recml_amd.kv_read(got, table.cuda(), zero, count=n, dtype=F32), (k, v)):
    assert torch.equal(r.cpu().double(), R.stored(x, 8))
  assert got.k[69_999].any() and got.k[3].any() and not got.k[69_997].any() and not got.k[0].any()
  out = recml_amd.cached_attention(q.cuda(), got, table.cuda(), torch.tensor([n]).cuda(), max_len=n)
  want = R.attention(q[0], R.stored(k, 8)[0], R.stored(v, 8)[0], length=n, held=torch.ones(n, dtype=torch.bool), max_len=n)
  assert ((out[0].cpu().double() - want[0]).abs() <= R.attention_tolerance(*want, n, F32)).all()


def test_calls_from_two_threads(gpu):
  """Two threads, each on a stream of its own, reading one cache."""
  import threading
  c = [_case(B=2, H=2, d=64, bits=4, page=64, lengths=[700, 90], counts=[1, 1], max_len=700, dtype=BF16, packed=False, seed=8, ts="heads",
             bucket_size=size) for size in (0.301, 0.5)]
  want = [recml_amd.cached_attention(x[1], x[0], x[2], x[3], **x[4]) for x in c]
  torch.cuda.synchronize()
  bad = []
  def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
      outs = [recml_amd.cached_attention(c[i][1], c[i][0], c[i][2], c[i][3], **c[i][4]) for _ in range(50)]
      torch.cuda.current_stream().synchronize()
      if not all(torch.equal(o, want[i]) for o in outs):
        bad.append(i)
  threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert not bad


def test_numbers_past_32_bits_and_outputs_that_overlap_are_refused(gpu):
  """Counts that the kernels' 32 bits would cut off, an output whose rows share memory, an output that wants a gradient."""
  got, rows, table, lens, call, want, counts = _case(B=2, H=2, d=64, bits=8, page=64, lengths=[130, 20], counts=[2, 2], max_len=130, dtype=BF16,
                                                     packed=False, seed=9)
  flat, offsets = rows.reshape(4, 2, 64), torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
  for change in (dict(max_len=2**32 + 130), dict(max_len=2**30 + 1), dict(out=rows[:, :1].expand_as(rows)), dict(out=rows.clone().requires_grad_(True))):
    with pytest.raises(ValueError):
      recml_amd.cached_attention(rows, got, table, lens, **dict(call, **change))
  for many in (2**32 + 2, 2**30 + 1, -1):
    with pytest.raises(ValueError, match="max_new"):
      recml_amd.cached_attention(flat, got, table, lens, **dict(call, offsets=offsets, max_new=many))
    with pytest.raises(ValueError, match="max_new"):
      recml_amd.kv_write(got, flat, flat, table, lens, offsets=offsets, max_new=many)
    with pytest.raises(ValueError):
      recml_amd.kv_read(got, table, lens, offsets=offsets, max_new=many, total=4)
    with pytest.raises(ValueError):
      recml_amd.kv_read(got, table, lens, count=many)
