"""Products of rows in 8 bits where their values are the smallest that the format has, against 64 bits."""

import pytest
import torch

import recml_amd
from tests import rows8_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# one size for each kernel: few rows, tiles of 64, with four sets of waves, of 128, with two sets, of 256 or their like (turns), rows in registers
SIZES = [(3, 300, 40), (16, 640, 200), (100, 300, 300), (64, 4096, 520), (4000, 300, 2000), (400, 8192, 700), (4096, 4096, 4096), (9000, 200, 1600)]


def _rows(codes, exponent, width, gpu):
  """Rows of these codes (in the first columns of their last block) under one exponent byte."""
  blocks = -(-width // 128)
  all_ = torch.zeros((codes.shape[0], 128 * blocks), dtype=torch.uint8)
  all_[:, 128 * (blocks - 1) : 128 * (blocks - 1) + codes.shape[1]] = codes
  exponents = torch.full((-(-blocks // 4), codes.shape[0], 4), exponent, dtype=torch.uint8)
  return recml_amd.Rows8(all_.to(gpu), exponents.to(gpu), width)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", SIZES)
@pytest.mark.parametrize("exponent", [1, 2, 3, 4, 246])
def test_one_value_times_a_power(gpu, exponent, rows, depth, cols, dtype):
  """Every code under the smallest exponents times a large power, and the other way round: exact in bf16 (a code has four bits), and for fp32
  results but for what the smallest two exponents have below bf16's least, 2^-133: the nearest multiple of it, ties to the even one."""
  codes = torch.arange(127, dtype=torch.uint8)[:, None].repeat(-(-rows // 127), 1)[:rows]
  x = _rows(codes, exponent, depth, gpu)
  w = _rows(torch.full((cols, 1), 56, dtype=torch.uint8), 127 + (100 if exponent < 100 else -100), depth, gpu)      # 56: 1.0
  values = torch.tensor(R.E4M3, dtype=torch.float64)[codes[:, 0].long()] * 2.0 ** (exponent - 127)
  if dtype == F32:
    values = torch.round(values * 2.0**133) * 2.0**-133
  want = (values * 2.0 ** (100 if exponent < 100 else -100))[:, None].expand(rows, cols).to(dtype)
  assert torch.equal(recml_amd.gemm_rows8(x, w, dtype=dtype).cpu(), want)
  assert torch.equal(recml_amd.gemm_rows8(w, x, dtype=dtype).cpu(), want.t())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", [(9, 300, 70), (130, 520, 300)])
def test_small_rows_times_large_ones(gpu, rows, depth, cols, dtype):
  """For fp32 results a value under 2^-133 is off by at most half of that."""
  g = torch.Generator().manual_seed(rows)
  x = recml_amd.quantize_rows((torch.randn((rows, depth), generator=g, dtype=torch.float64) * 2.0**-128).to(F32).to(gpu))
  w = recml_amd.quantize_rows((torch.randn((cols, depth), generator=g) * 2.0**100).to(gpu))
  a, b = R.values(x.codes, x.exponents, depth), R.values(w.codes, w.exponents, depth)
  assert (x.exponents[0, :, 0] <= 2).all()
  y, before, sizes = R.product(a, b, None, None, False)
  off = R.product_off(y, before, sizes, depth, dtype, False)
  if dtype == F32:
    off = off + 2.0**-134 * b.abs().sum(1)[None, :]
  assert float(((recml_amd.gemm_rows8(x, w, dtype=dtype).cpu().double() - y).abs() - off).max()) <= 0


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype,last", [(BF16, 59), (F32, 63)])
def test_the_largest_rows_that_have_a_norm(gpu, dtype, last, rms):
  """256 values of 2^p of both signs, whose norm is their sign: the sum of their squares has to lie within fp32 for rows in bf16, its mean for
  rows in fp32; past that it counts as infinite and the row as zeros."""
  signs = torch.where(torch.randperm(256, generator=torch.Generator().manual_seed(1)) < 128, 1.0, -1.0)
  gamma = torch.ones(256, dtype=dtype, device=gpu)
  for p in (last, last + 1, 100):
    x = (signs * 2.0**p).to(dtype)[None].to(gpu)
    want = signs if p == last else torch.zeros(256)
    assert torch.equal(recml_amd.norm_rows8(x, gamma, rms=rms).values(F32)[0].cpu(), want), p


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype,first", [(BF16, -63), (F32, -126)])
def test_the_smallest_rows_that_have_a_norm_without_eps(gpu, dtype, first, rms):
  """The mean of their squares has to be a normal number of the type that statistics are in: fp32 for rows in bf16, 64 bits for rows in fp32."""
  signs = torch.where(torch.randperm(256, generator=torch.Generator().manual_seed(1)) < 128, 1.0, -1.0)
  gamma = torch.ones(256, dtype=dtype, device=gpu)
  x = (signs * 2.0**first).to(dtype)[None].to(gpu)
  assert torch.equal(recml_amd.norm_rows8(x, gamma, eps=0.0, rms=rms).values(F32)[0].cpu(), signs)
