"""Rows in 8 bits: quantising, norms into them, what they stand for, and their products, against 64 bits."""

import ctypes as C
import threading

import pytest
import torch

import recml_amd
from recml_amd import _lib_rows8
from tests import rows8_reference as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _rows(rows, width, dtype, seed, spread=1.0):
  g = _gen(seed)
  return (torch.randn((rows, width), generator=g) * torch.exp(spread * torch.randn((rows, width), generator=g))).to(dtype)


def _same(rows, x):
  codes, exponents = R.quantised(x)
  assert rows.rows == x.shape[0] and rows.width == x.shape[1]
  assert torch.equal(rows.exponents.cpu(), exponents)
  assert torch.equal(rows.codes.cpu(), codes)


WIDTHS = [1, 2, 7, 8, 9, 63, 64, 120, 127, 128, 129, 200, 255, 256, 257, 511, 512, 513, 520, 640, 1000, 1001, 1024, 1025, 2047, 2048, 2049, 4100, 8192, 8193, 32768]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantised_exactly(gpu, width, dtype):
  x = _rows(3, width, dtype, width, 2.0)
  rows = recml_amd.quantize_rows(x.to(gpu))
  _same(rows, x)
  want = R.values(rows.codes, rows.exponents, width)
  assert torch.equal(rows.values(F32).cpu(), want.to(F32))
  assert torch.equal(rows.values().cpu(), want.to(BF16))


@pytest.mark.parametrize("count", [0, 1, 2, 5, 64, 300])
def test_quantised_row_counts(gpu, count):
  for width in (24, 200, 500, 900, 3000):
    x = _rows(count, width, BF16, count)
    _same(recml_amd.quantize_rows(x.to(gpu)), x)


def test_quantised_at_the_borders(gpu):
  """Every border between codes, both sides of it, the blocks' own borders, zeros of both signs, the smallest and largest values."""
  levels = torch.tensor(R.E4M3, dtype=torch.float64)
  middles = (levels[1:] + levels[:-1]) / 2
  around = torch.cat([middles, middles * (1 + 2.0**-23), middles * (1 - 2.0**-23), levels, torch.tensor([448.0, 463.9, 464.0])])
  rows = [torch.nn.functional.pad(around[i : i + 127], (1, 0), value=448.0) for i in range(0, len(around), 127)]
  x = torch.nn.utils.rnn.pad_sequence(rows, batch_first=True)
  x = torch.cat([x, -x, x * 2.0**-100, x * 2.0**100])
  tops = torch.zeros((12, 128), dtype=torch.float64)
  for i, top in enumerate((464.0, 464.0 * (1 + 2.0**-23), 232.0, 232.0 * (1 + 2.0**-23), 448.0, 2.0**-149, 2.0**-126, 1.9 * 2.0**-127, 3.4028234663852886e38, 1.8125 * 2.0**127, -0.0, 0.0)):
    tops[i, 5] = top
  x = torch.cat([x, torch.nn.functional.pad(tops, (0, x.shape[1] - 128))]).to(F32)
  _same(recml_amd.quantize_rows(x.to(gpu)), x)
  x = x.to(BF16)
  _same(recml_amd.quantize_rows(x.to(gpu)), x)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_blocks_that_are_not_finite(gpu, dtype):
  x = _rows(4, 700, dtype, 1)
  x[0, 130], x[1, 699], x[2, 0], x[2, 300] = float("nan"), float("inf"), float("-inf"), float("nan")
  rows = recml_amd.quantize_rows(x.to(gpu))
  _same(rows, x)
  got = torch.isnan(rows.values().cpu())
  want = torch.zeros_like(got)
  want[0, 128:256] = want[1, 640:] = want[2, :128] = want[2, 256:384] = True
  assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(gpu, dtype):
  """Slices, transposes, expanded and misaligned rows, more axes: the rows that a contiguous tensor has."""
  big = _rows(24, 264, dtype, 2).to(gpu)
  for x in (big[:, 8:136], big[:, 3:120], big[::2, :128], big.t(), big[5:6].expand(7, 264), big.reshape(2, 3, 4, 264)[:, 1:], big.reshape(4, 6, 264).transpose(0, 1),
            big.reshape(24, 2, 132)[:, 1], big[0], big.reshape(-1)[1:1 + 20 * 200].view(20, 200)):
    rows = recml_amd.quantize_rows(x)
    _same(rows, x.reshape(-1, x.shape[-1]).cpu())


NORMS = [(1, 1), (5, 3), (3, 8), (7, 64), (4, 100), (130, 128), (3, 129), (9, 250), (6, 512), (3, 520), (5, 777), (2, 1000), (3, 1024), (2, 1500), (2, 2048), (2, 3001),
         (2, 8192), (2, 10000)]
NORMS += [(33, 40), (17, 41), (9, 136), (9, 256), (4, 1001), (3, 2047), (3, 4096), (3, 4095), (2, 8191), (2, 16384), (2, 32767), (2, 32768), (130, 5), (300, 9), (129, 16), (70, 17), (65, 31), (66, 32)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,width", NORMS)
def test_norm(gpu, rows, width, kind, dtype):
  g = _gen(rows * width)
  new = lambda *shape, std=1.0, mean=0.0: (torch.randn(shape, generator=g) * std + mean).to(dtype)
  x, other, u = new(rows, width, mean=0.3), new(rows, width), new(rows, width, std=0.5)
  gamma, beta = new(width, std=0.2, mean=1.0), new(width, std=0.1)
  for add in (None, other):
    for gate in (None, u):
      for b in (None, beta):
        put = lambda t: None if t is None else t.to(gpu)
        got = recml_amd.norm_rows8(put(x), put(gamma), put(b), 1e-5, gate=put(gate), add=put(add), rms=kind == "rms")
        s = x
        if add is not None:
          got, total = got
          s = (x.float() + add.float()).to(dtype)
          assert torch.equal(total.cpu(), s)
        R.check_stored(got, *R.norm(s, gamma, b, 1e-5, gate, kind))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_of_slices(gpu, dtype):
  """The gate as a slice of a fused projection, x and the residual as slices of their own, on [B, n, W]."""
  g = _gen(5)
  new = lambda *shape: torch.randn(shape, generator=g).to(dtype)
  wide, other, x = new(3, 4, 4, 96), new(3, 4, 100), new(3, 4, 104)
  gamma, beta = new(96), new(96)
  for at in (0, 1):
    s, a, u = x[..., 8 * at : 8 * at + 96], other[..., at : at + 96], wide[:, :, 2]
    put = lambda base, view: base.to(gpu).as_strided(view.shape, view.stride(), view.storage_offset())
    got, total = recml_amd.norm_rows8(put(x, s), gamma.to(gpu), beta.to(gpu), gate=put(wide, u), add=put(other, a))
    s = (s.float() + a.float()).to(dtype)
    assert torch.equal(total.cpu(), s)
    R.check_stored(got, *R.norm(s.reshape(-1, 96), gamma, beta, 1e-6, u.reshape(-1, 96), "layer"))


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,width", [(4000, 40), (700, 999), (300, 1384), (120, 4097), (40, 16000)])
def test_codes_of_rows_in_32_bits(gpu, rows, width, kind):
  """Their values are taken in 64 bits, so that the roundings which norm() counts are 2^29 times smaller (twice that with its own)."""
  g = _gen(rows + width)
  x, gate = torch.randn((rows, width), generator=g) * 2 + 0.5, torch.randn((rows, width), generator=g)
  gamma, beta = torch.randn(width, generator=g) + 1.0, torch.randn(width, generator=g) * 0.2 if kind == "layer" else None
  got = recml_amd.norm_rows8(x.to(gpu), gamma.to(gpu), None if beta is None else beta.to(gpu), 2.0**-20, rms=kind == "rms", gate=gate.to(gpu))
  y, off = R.norm(x, gamma, beta, 2.0**-20, gate, kind)
  R.check_stored(got, y, off * 2.0**-28)


def test_norm_of_what_has_none(gpu):
  """Rows of one value, constant rows, rows with a NaN or an infinity, and sums past fp32."""
  x = torch.zeros((6, 200))
  x[1], x[2, 7], x[3, 9], x[4], x[5] = 3.0, float("nan"), float("inf"), 1e30, torch.linspace(-1, 1, 200)
  gamma = torch.ones(200, device=gpu)
  for rms in (False, True):
    got = recml_amd.norm_rows8(x.to(gpu), gamma, None, 1e-6, rms=rms).values(F32).cpu()
    # (an infinity's mean is one, and no difference from it a number; under the root mean square of infinity all else is 0)
    assert torch.isnan(got[2]).all() and torch.isnan(got[3, :128]).all() and (torch.isnan(got[3]).all() if not rms else (got[3, 128:] == 0).all())
    assert (got[0] == 0).all() and torch.isfinite(got[5]).all()
    assert (got[1] == 0).all() if not rms else ((got[1] - 1).abs() <= 2.0**-4).all()
    assert (got[4] == 0).all()                                   # (the squares are past fp32: rstd is 0)


PRODUCTS = [(1, 1, 1), (1, 128, 64), (2, 129, 7), (31, 64, 33), (32, 128, 32), (33, 200, 31), (5, 300, 77), (64, 128, 65), (65, 513, 64), (100, 512, 300), (128, 1000, 256), (129, 640, 513),
            (300, 384, 130), (17, 2000, 1000), (257, 100, 257), (1, 4100, 48), (70, 8192, 40), (129, 2600, 513)]


def _check_product(got, x, w, bias, residual, activation, dtype):
  y, before, size = R.product(R.values(x.codes, x.exponents, x.width), R.values(w.codes, w.exponents, w.width), bias, residual, activation)
  off = R.product_off(y, before, size, x.width, dtype, activation)
  assert got.dtype == dtype and tuple(got.shape) == tuple(y.shape)
  far = (got.cpu().double() - y).abs() - off
  assert float(far.max()) <= 0, (float(far.max()), float(((got.cpu().double() - y).abs() / off).max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", PRODUCTS)
def test_product(gpu, rows, depth, cols, dtype):
  g = _gen(rows + depth + cols)
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n + depth, 1.0).to(gpu)) for n in (rows, cols))
  bias, residual = torch.randn(cols, generator=g).to(dtype), torch.randn((rows, cols), generator=g).to(dtype)
  for b, c, act in ((None, None, False), (bias, None, True), (None, residual, False), (bias, residual, True)):
    got = recml_amd.gemm_rows8(x, w, None if b is None else b.to(gpu), act, residual=None if c is None else c.to(gpu), dtype=dtype)
    _check_product(got, x, w, b, c, act, dtype)


LARGE = [(700, 512, 2048), (2100, 256, 1030), (9000, 200, 520), (64, 512, 9000), (16, 1024, 5000), (3000, 1024, 4096),
         (4000, 1500, 4000), (4000, 650, 4090), (700, 4200, 3700), (200, 4000, 4100), (1000, 4200, 4000)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", LARGE)
def test_large_product(gpu, rows, depth, cols, dtype):
  """The tiles of large calls, against 64 bits on the GPU."""
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n, 0.5).to(gpu)) for n in (rows, cols))
  residual = torch.randn((rows, cols), generator=_gen(1)).to(dtype).to(gpu)
  a, b = (R.values(t.codes, t.exponents, depth).to(gpu) for t in (x, w))
  for c in (None, residual):
    y, before, size = R.product(a, b.contiguous(), None, c, False)
    off = R.product_off(y, before, size, depth, dtype, False)
    got = recml_amd.gemm_rows8(x, w, residual=c, dtype=dtype)
    assert float(((got.double() - y).abs() - off).max()) <= 0


@pytest.mark.parametrize("how", ["plain", "silu", "added"])
@pytest.mark.parametrize("depth", [40, 256, 300, 512, 640, 700, 896, 1024])
def test_many_outputs_of_short_contractions(gpu, depth, how):
  """Rows kept in registers: every number of blocks, a last tile that is not whole, runs that begin and end inside a tile."""
  rows, cols = 256 * 11 - 37, 64 * 75
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n, 0.5).to(gpu)) for n in (rows, cols))
  c = torch.randn((rows, cols + 8), generator=_gen(depth)).to(BF16).to(gpu)[:, :cols] if how == "added" else None
  got = recml_amd.gemm_rows8(x, w, None, how == "silu", residual=c)
  y, before, sizes = R.product(R.values(x.codes, x.exponents, depth).to(gpu), R.values(w.codes, w.exponents, depth).to(gpu), None, c, how == "silu")
  assert float(((got.double() - y).abs() - R.product_off(y, before, sizes, depth, BF16, how == "silu")).max()) <= 0
  assert torch.equal(got, recml_amd.gemm_rows8(x, w, None, how == "silu", residual=c))
  if c is None:                                # (with a bias the call goes by tiles, whose sums are the same)
    assert torch.equal(got, recml_amd.gemm_rows8(x, w, torch.zeros(cols, dtype=BF16, device=gpu), how == "silu"))


@pytest.mark.parametrize("depth", [128, 200, 384, 512, 600, 768, 800, 1000])
def test_many_sums_of_short_contractions(gpu, depth):
  """As above where something is added, in as many outputs as that takes."""
  rows, cols = 256 * 17 - 37, 64 * 77
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n, 0.5).to(gpu)) for n in (rows, cols))
  c = torch.randn((rows, cols + 8), generator=_gen(depth)).to(BF16).to(gpu)[:, :cols]
  got = recml_amd.gemm_rows8(x, w, residual=c)
  y, before, sizes = R.product(R.values(x.codes, x.exponents, depth).to(gpu), R.values(w.codes, w.exponents, depth).to(gpu), None, c, False)
  assert float(((got.double() - y).abs() - R.product_off(y, before, sizes, depth, BF16, False)).max()) <= 0
  assert torch.equal(got, recml_amd.gemm_rows8(x, w, residual=c))


@pytest.mark.parametrize("how", ["bias", "bias silu", "added silu", "added bias"])
@pytest.mark.parametrize("depth", [128, 200, 384, 512, 600, 768, 800, 1000])
def test_many_outputs_of_short_contractions_with_a_bias(gpu, depth, how):
  """A bias that starts between two 16-byte pieces among them."""
  rows, cols = 256 * 17 - 37, 64 * 77
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n, 0.5).to(gpu)) for n in (rows, cols))
  b = torch.randn(cols + 1, generator=_gen(depth)).to(BF16).to(gpu)[1:] if "bias" in how else None
  c = torch.randn((rows, cols), generator=_gen(depth + 1)).to(BF16).to(gpu) if "added" in how else None
  got = recml_amd.gemm_rows8(x, w, b, "silu" in how, residual=c)
  y, before, sizes = R.product(R.values(x.codes, x.exponents, depth).to(gpu), R.values(w.codes, w.exponents, depth).to(gpu), b, c, "silu" in how)
  assert float(((got.double() - y).abs() - R.product_off(y, before, sizes, depth, BF16, "silu" in how)).max()) <= 0
  assert torch.equal(got, recml_amd.gemm_rows8(x, w, b, "silu" in how, residual=c))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", [(1, 128, 24), (20, 300, 40), (50, 300, 72), (300, 200, 136), (2000, 200, 1032), (7000, 200, 2120), (2779, 500, 4800), (130, 2600, 520), (700, 4200, 3704)])
def test_leaves_what_is_not_its_own(gpu, rows, depth, cols, dtype):
  """Rows with a stride of their own in the middle of a buffer: what stands between, before and behind them stays."""
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n, 0.5).to(gpu)) for n in (rows, cols))
  stride, unit = cols + 8, 16
  buffer = torch.full((unit + rows * stride + unit,), 7.0, dtype=dtype, device=gpu)
  a = _lib_rows8.HstuRows8GemmArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_rows8.ABI_VERSION
  x._fill(a.x)
  w._fill(a.w)
  a.dtype, a.out, a.out_stride = (_lib_rows8.FP32 if dtype == F32 else _lib_rows8.BF16), buffer[unit:].data_ptr(), stride
  assert _lib_rows8.load().hstu_rows8_gemm(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
  torch.cuda.synchronize()
  assert (buffer[:unit] == 7).all() and (buffer[-unit:] == 7).all()
  body = buffer[unit:-unit].view(rows, stride)
  assert (body[:, cols:] == 7).all()
  assert torch.equal(body[:, :cols], recml_amd.gemm_rows8(x, w, dtype=dtype))


def _arguments(kind, dtype):
  a = kind()
  a.struct_size, a.version, a.dtype = C.sizeof(a), _lib_rows8.ABI_VERSION, _lib_rows8.FP32 if dtype == F32 else _lib_rows8.BF16
  return a, C.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", [(8, 512, 64), (100, 300, 77), (64, 4096, 520), (257, 640, 1000), (256 * 17 - 37, 384, 64 * 77), (4096, 1500, 4096), (1000, 4200, 1000)])
def test_product_added_in_place(gpu, rows, depth, cols, dtype):
  x, w = (recml_amd.quantize_rows(_rows(n, depth, F32, n, 0.5).to(gpu)) for n in (rows, cols))
  out = torch.randn((rows, cols), generator=_gen(rows), dtype=F32).to(dtype).to(gpu)
  want = recml_amd.gemm_rows8(x, w, residual=out, dtype=dtype)
  a, stream = _arguments(_lib_rows8.HstuRows8GemmArgs, dtype)
  x._fill(a.x)
  w._fill(a.w)
  a.out = a.c = out.data_ptr()
  a.out_stride = a.c_stride = cols
  assert _lib_rows8.load().hstu_rows8_gemm(C.byref(a), stream) == 0
  assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", [3, 64, 999, 2048, 5000, 16001])
@pytest.mark.parametrize("onto", ["x", "add"])
def test_norm_of_a_sum_in_place(gpu, width, onto, dtype):
  g = _gen(width)
  new = lambda *shape: torch.randn(shape, generator=g).to(dtype).to(gpu)
  x, add, gate, gamma = new(40, width), new(40, width), new(40, width), new(width)
  want, total = recml_amd.norm_rows8(x, gamma, gate=gate, add=add)
  got = recml_amd.Rows8._empty(40, width, x.device)
  a, stream = _arguments(_lib_rows8.HstuRows8NormArgs, dtype)
  got._fill(a.rows)
  a.norm, a.eps = _lib_rows8.LAYER, 1e-6
  a.x, a.add, a.gate, a.gamma = x.data_ptr(), add.data_ptr(), gate.data_ptr(), gamma.data_ptr()
  a.x_stride = a.add_stride = a.gate_stride = a.sum_stride = width
  put = x if onto == "x" else add
  a.sum = put.data_ptr()
  assert _lib_rows8.load().hstu_rows8_norm(C.byref(a), stream) == 0
  assert torch.equal(put, total) and torch.equal(got.codes, want.codes) and torch.equal(got.exponents, want.exponents)


def test_first_calls_in_a_capture(gpu):
  """A graph that no eager call of these sizes came before, replayed between eager work."""
  g = _gen(21)
  x, gamma = torch.randn((130, 4300), generator=g).to(BF16).to(gpu), torch.ones(4300, dtype=BF16, device=gpu)
  w = recml_amd.quantize_rows(torch.randn((1030, 4300), generator=g).to(gpu))
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    kept = recml_amd.gemm_rows8(recml_amd.norm_rows8(x, gamma), w)
  for i in range(3):
    x.copy_(torch.randn((130, 4300), generator=g))
    graph.replay()
    assert torch.equal(kept, recml_amd.gemm_rows8(recml_amd.norm_rows8(x, gamma), w)), i


def test_sums_in_fp32(gpu):
  """An fp32 result has fp32's precision: independent roundings of partial sums, each at most half a step of the sum of the magnitudes, add up to
  sqrt(depth) of that in the mean square."""
  depth = 4096
  x, w = (recml_amd.quantize_rows(_rows(200, depth, F32, s, 0.5).to(gpu)) for s in (1, 2))
  y, _, size = R.product(R.values(x.codes, x.exponents, depth), R.values(w.codes, w.exponents, depth), None, None, False)
  err = recml_amd.gemm_rows8(x, w, dtype=F32).cpu().double() - y
  assert float(err.square().mean().sqrt()) <= depth**0.5 * R.STEP * float(size[0].square().mean().sqrt())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_products_of_powers(gpu, dtype):
  """Powers of two at all ends of the range: exact, and past it infinite or, under it, zero."""
  powers = [-126, -120, -64, -30, -1, 0, 1, 30, 64, 119, 127]
  x = torch.stack([torch.full((256,), 2.0**p) for p in powers])
  rows = recml_amd.quantize_rows(x.to(gpu))
  got = recml_amd.gemm_rows8(rows, rows, dtype=dtype).cpu().double()
  for i, a in enumerate(powers):
    for j, b in enumerate(powers):
      want = 256 * 2.0 ** (a + b)
      if a + b + 8 > 127:
        assert torch.isinf(got[i, j]), (a, b)
      elif a + b + 8 >= -126:
        assert float(got[i, j]) == want, (a, b)
      else:
        assert 0 <= float(got[i, j]) <= want, (a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product_of_what_is_not_finite(gpu, dtype):
  x, w = _rows(40, 300, F32, 1), _rows(70, 300, F32, 2)
  x[3, 290], x[7] = float("nan"), 0.0
  w[5, 10], w[69, 200] = float("inf"), float("nan")
  got = recml_amd.gemm_rows8(*(recml_amd.quantize_rows(t.to(gpu)) for t in (x, w)), dtype=dtype).cpu()
  want = torch.zeros((40, 70), dtype=torch.bool)
  want[3] = want[:, 5] = want[:, 69] = True
  assert torch.equal(torch.isnan(got), want)
  assert (got[7][~want[7]] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product_layouts(gpu, dtype):
  """Residuals as slices, transposes and expanded rows, bias misaligned: what contiguous ones give."""
  x, w = (recml_amd.quantize_rows(_rows(n, 160, F32, n).to(gpu)) for n in (40, 56))
  big, long = torch.randn((80, 120), generator=_gen(3)).to(dtype).to(gpu), torch.randn(61, generator=_gen(4)).to(dtype).to(gpu)
  for c in (big[:40, :56], big[:40, 3:59], big[::2, 8:64], big[:56, :40].t(), big[3:4, :56].expand(40, 56), big[:40, :1].expand(40, 56)):
    for b in (long[:56], long[1:57], long[5:6].expand(56), long[:56].reshape(7, 8)):
      got = recml_amd.gemm_rows8(x, w, b, True, residual=c, dtype=dtype)
      assert torch.equal(got, recml_amd.gemm_rows8(x, w, b.reshape(-1).clone(), True, residual=c.clone(memory_format=torch.contiguous_format), dtype=dtype))
      _check_product(got, x, w, b.cpu().reshape(-1), c.cpu(), True, dtype)


def test_nothing_to_do(gpu):
  empty, some = recml_amd.quantize_rows(torch.zeros((0, 40), device=gpu)), recml_amd.quantize_rows(torch.ones((3, 40), device=gpu))
  assert tuple(recml_amd.gemm_rows8(empty, some).shape) == (0, 3) and tuple(recml_amd.gemm_rows8(some, empty).shape) == (3, 0)
  assert tuple(empty.values().shape) == (0, 40)
  rows, total = recml_amd.norm_rows8(torch.zeros((2, 0, 40), device=gpu), torch.ones(40, device=gpu), add=torch.zeros((2, 0, 40), device=gpu))
  assert rows.rows == 0 and tuple(total.shape) == (2, 0, 40)


def _steps(x, attn, gammas, betas, w, w_out, H=4):
  rows, total = recml_amd.norm_rows8(x, gammas[0], betas[0], add=attn)
  uqkv = recml_amd.gemm_rows8(rows, w, None, True, dtype=x.dtype)
  W = x.shape[1]
  gated = recml_amd.norm_rows8(attn, gammas[1], betas[1], gate=uqkv[:, :W])
  return rows, total, uqkv, gated, recml_amd.gemm_rows8(gated, w_out, residual=total, dtype=x.dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,width", [(1, 64), (50, 136), (333, 512)])
def test_a_run_of_steps(gpu, tokens, width, dtype):
  """A block's steps one behind the other, each against 64 bits on what the one before handed on."""
  g = _gen(tokens)
  new = lambda *shape, std=1.0: (torch.randn(shape, generator=g) * std).to(dtype).to(gpu)
  x, attn = new(tokens, width), new(tokens, width, std=0.1)
  gammas, betas = (1 + new(2, width, std=0.1), new(2, width, std=0.1))
  w, w_out = (recml_amd.quantize_rows(new(n, width, std=width**-0.5)) for n in (4 * width, width))
  rows, total, uqkv, gated, out = _steps(x, attn, gammas, betas, w, w_out)
  R.check_stored(rows, *R.norm(total.cpu(), gammas[0].cpu(), betas[0].cpu(), 1e-6, None, "layer"))
  _check_product(uqkv, rows, w, None, None, True, dtype)
  R.check_stored(gated, *R.norm(attn.cpu(), gammas[1].cpu(), betas[1].cpu(), 1e-6, uqkv[:, :width].cpu(), "layer"))
  _check_product(out, gated, w_out, None, total.cpu(), False, dtype)


def test_captured_and_replayed(gpu):
  g = _gen(9)
  new = lambda *shape: torch.randn(shape, generator=g).to(BF16).to(gpu)
  x, attn, gammas, betas = new(70, 264), new(70, 264), new(2, 264), new(2, 264)
  w, w_out = recml_amd.quantize_rows(new(4 * 264, 264)), recml_amd.quantize_rows(new(264, 264))
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    _steps(x, attn, gammas, betas, w, w_out)
  side.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    kept = _steps(x, attn, gammas, betas, w, w_out)
  for i in range(4):
    x.copy_(new(70, 264))
    attn.copy_(new(70, 264))
    want = _steps(x, attn, gammas, betas, w, w_out)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(kept, want):
      a, b = (t.codes if isinstance(t, recml_amd.Rows8) else t for t in (a, b))
      assert torch.equal(a, b), i


def test_two_threads_on_streams_of_their_own(gpu):
  g = _gen(11)
  new = lambda *shape: torch.randn(shape, generator=g).to(BF16).to(gpu)
  x, gamma, w = new(2, 300, 512), new(512), recml_amd.quantize_rows(new(640, 512))
  want = [recml_amd.gemm_rows8(recml_amd.norm_rows8(x[i], gamma), w) for i in range(2)]
  torch.cuda.synchronize()
  got = [[], []]

  def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
      for _ in range(20):
        got[i].append(recml_amd.gemm_rows8(recml_amd.norm_rows8(x[i], gamma), w))
      torch.cuda.current_stream().synchronize()

  threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  for i in range(2):
    assert len(got[i]) == 20 and all(torch.equal(y, want[i]) for y in got[i])


def test_the_same_bits_whatever_stands_beside(gpu):
  """A row's result does not depend on the rows beside it, as long as the call takes the same kernel; runs agree bit by bit."""
  x, w = _rows(40, 300, BF16, 1).to(gpu), recml_amd.quantize_rows(_rows(50, 300, BF16, 2).to(gpu))
  all_ = recml_amd.gemm_rows8(recml_amd.quantize_rows(x), w)
  assert torch.equal(all_, recml_amd.gemm_rows8(recml_amd.quantize_rows(x), w))
  other = x.clone()
  other[:20] = float("nan")
  assert torch.equal(recml_amd.gemm_rows8(recml_amd.quantize_rows(other), w)[20:], all_[20:])


def test_offsets_past_32_bits(gpu):
  """A table of 9 million rows of 512: more than 2^32 bytes of codes."""
  rows = 9_000_000
  x = torch.zeros((rows, 512), dtype=BF16, device=gpu)
  tail = _rows(300, 512, BF16, 3).to(gpu)
  x[-300:] = tail
  kept = recml_amd.quantize_rows(x)
  del x
  small = recml_amd.quantize_rows(tail)
  assert torch.equal(kept.codes[-300:], small.codes) and torch.equal(kept.exponents[:, -300:], small.exponents)
  assert torch.equal(kept.values()[-300:], small.values())
  probe = recml_amd.quantize_rows(_rows(3, 512, BF16, 4).to(gpu))
  got = recml_amd.gemm_rows8(probe, kept)
  assert not got[:, :-300].any()
  y, before, size = R.product(R.values(probe.codes, probe.exponents, 512), R.values(small.codes, small.exponents, 512), None, None, False)
  assert float(((got[:, -300:].cpu().double() - y).abs() - R.product_off(y, before, size, 512, BF16, False)).max()) <= 0
  got = recml_amd.gemm_rows8(kept, probe)
  assert not got[:-300].any()
  assert float(((got[-300:].cpu().double() - y.t()).abs() - R.product_off(y, before, size, 512, BF16, False).t()).max()) <= 0
