"""Products of rows in 8 bits, one size for each of their kernels: blocks that are not numbers, and kernels against each other bit by bit."""

import pytest
import torch

import recml_amd

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# few rows, more of them, tiles of 64, with four sets of waves, of 128, with two sets, of 256 (turns), rows in registers of 2 and of 8 blocks
SIZES = [(3, 700, 40), (30, 640, 200), (100, 600, 300), (64, 4096, 520), (4000, 600, 2000), (400, 8192, 700), (4096, 4096, 4096), (9000, 200, 1600), (9000, 1000, 1600)]


def _rows(rows, width, seed, gpu):
  return torch.randn((rows, width), generator=torch.Generator(gpu).manual_seed(seed), device=gpu)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,depth,cols", SIZES)
@pytest.mark.parametrize("how", ["plain", "silu", "bias", "added"])
def test_blocks_that_are_not_numbers(gpu, rows, depth, cols, how, dtype):
  """One in each place of a group of four blocks, in both operands, first and last rows among them: NaN where they take part, and elsewhere
  the bits that the call has without them."""
  x, w = _rows(rows, depth, 1, gpu), _rows(cols, depth, 2, gpu)
  bias = _rows(1, cols, 3, gpu)[0].to(dtype) if how == "bias" else None
  c = _rows(rows, cols, 4, gpu).to(dtype) if how == "added" else None
  call = lambda: recml_amd.gemm_rows8(recml_amd.quantize_rows(x), recml_amd.quantize_rows(w), bias, how == "silu", residual=c, dtype=dtype)
  clean = call()
  assert torch.isfinite(clean).all()
  want_x, want_w = torch.zeros(rows, dtype=torch.bool), torch.zeros(cols, dtype=torch.bool)
  for i, value in enumerate((float("nan"), float("inf"), float("-inf"), float("nan"), float("inf"), float("nan"))):
    at = min(128 * i + 5 * i, depth - 1)                     # (the last one in the row's last value where it is short)
    r, n = (0, rows - 1, rows // 2, rows // 3, rows // 5, rows // 7)[i], (cols - 1, 0, cols // 2, cols // 3, cols // 5, cols // 7)[i]
    x[r, at], w[n, at] = value, value
    want_x[r] = want_w[n] = True
  got = call()
  want = (want_x[:, None] | want_w[None, :]).to(gpu)
  assert torch.equal(torch.isnan(got), want)
  assert torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("how", ["plain", "silu"])
@pytest.mark.parametrize("depth", [40, 256, 300, 512, 640, 700, 896, 1024])
def test_rows_in_registers_have_the_tiles_bits(gpu, depth, how):
  """A call with a bias and rows to be added goes by tiles, whose sums are made in the same order: zeros of both leave the sums as they are."""
  rows, cols = 256 * 11 - 37, 64 * 75
  x, w = recml_amd.quantize_rows(_rows(rows, depth, depth, gpu)), recml_amd.quantize_rows(_rows(cols, depth, depth + 1, gpu))
  got = recml_amd.gemm_rows8(x, w, None, how == "silu")
  zeros = torch.zeros((rows, cols), dtype=BF16, device=gpu)
  assert torch.equal(got, recml_amd.gemm_rows8(x, w, zeros[0], how == "silu", residual=zeros))


@pytest.mark.parametrize("rows,depth,cols", SIZES)
def test_sums_of_ones(gpu, rows, depth, cols):
  """Ones of both signs, whose products and sums are exact in whatever order: every kernel has the sum's bits."""
  g = torch.Generator(gpu).manual_seed(rows)
  x, w = (torch.randint(0, 2, (n, depth), generator=g, device=gpu).float() * 2 - 1 for n in (rows, cols))
  want = (x.double() @ w.double().t()).float()
  for dtype in (BF16, F32):
    assert torch.equal(recml_amd.gemm_rows8(recml_amd.quantize_rows(x), recml_amd.quantize_rows(w), dtype=dtype), want.to(dtype))
