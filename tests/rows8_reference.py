"""The operators on rows in 8 bits in 64 bits, element by element from their definitions (CPU tensors in, CPU tensors out), and how far
fp32 arithmetic may be off."""

import math

import torch

E4M3 = [f / 512 for f in range(8)] + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8)][:119]
STEP = 2.0**-24


def exponent(top):
  """The smallest exponent (without its bias) under which `top` rounds to a code."""
  if not top > 0:
    return -126
  e = max(-126, math.frexp(top)[1] - 20)
  while top > 464.0 * 2.0**e and e < 119:
    e += 1
  return e


def quantised(x):
  """Rows [R, W] as (codes [R, 128 blocks], exponents [ceil(blocks / 4), R, 4])."""
  levels = torch.tensor(E4M3, dtype=torch.float64)
  R, W = x.shape
  blocks = -(-W // 128)
  codes = torch.zeros((R, 128 * blocks), dtype=torch.uint8)
  kept = torch.ones((R, -(-blocks // 4) * 4), dtype=torch.uint8)
  for r, row in enumerate(x.double()):
    for b in range(blocks):
      block = row[128 * b : 128 * b + 128]
      if not torch.isfinite(block).all():
        kept[r, b] = 255
        continue
      e = exponent(float(block.abs().max()))
      kept[r, b] = e + 127
      off = (block.abs()[:, None] / 2.0**e - levels[None, :]).abs()
      near = off == off.min(1, keepdim=True).values
      code = torch.where(near[:, 0::2].any(1), 2 * near[:, 0::2].int().argmax(1), 2 * near[:, 1::2].int().argmax(1) + 1)
      codes[r, 128 * b : 128 * b + len(block)] = (code + 128 * torch.signbit(block).long()).to(torch.uint8)
  return codes, kept.view(R, kept.shape[1] // 4, 4).transpose(0, 1).contiguous()


def values(codes, exponents, width):
  """What rows stand for, [R, width] in 64 bits."""
  c = codes.cpu().long()
  y = torch.tensor(E4M3 + [math.nan], dtype=torch.float64)[c % 128] * (1.0 - 2.0 * (c // 128))
  e = exponents.cpu().long().permute(1, 0, 2).flatten(1)[:, : c.shape[1] // 128]
  power = torch.where(e == 255, math.nan, torch.ldexp(torch.ones(1, dtype=torch.float64), e - 127))
  return (y * power.repeat_interleave(128, -1))[:, :width]


def norm(x, gamma, beta, eps, gate, kind):
  """gate * norm(x) of rows that are summed already, and how far fp32 may be off it.

  A sum over a row is chains of at most 16 additions and their tree: 48 roundings are more than any path through it has.  So the mean is off
  by 48 steps of the mean magnitude, the differences by that and one of their own, the variance (by Cauchy and Schwarz) by 48 steps of
  itself and twice the differences' over the deviation, rstd by half of that and 4 steps (its argument's two, its own two), and what
  follows by three roundings and the gate's."""
  x = x.double()
  mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros((x.shape[0], 1), dtype=torch.float64)
  d = x - mean
  var = (d * d).mean(-1, keepdim=True)
  rstd = 1 / torch.sqrt(var + eps)
  g = gamma.double()
  y = d * rstd * g + (0.0 if beta is None else beta.double())
  mean_off = 48 * STEP * x.abs().mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(mean)
  d_off = mean_off + STEP * d.abs()
  rel = 0.5 * (48 * STEP + 2 * (mean_off + STEP * var.sqrt()) * var.sqrt() / (var + eps)) + 4 * STEP
  off = g.abs() * rstd * (d_off + d.abs() * (rel + 3 * STEP)) + 2 * STEP * y.abs()
  if gate is not None:
    y, off = y * gate.double(), off * gate.double().abs() + STEP * (y * gate.double()).abs()
  return y, off


def check_stored(rows, y, off):
  """Whether rows in 8 bits are those of `y`, each value of which may be off by `off`: exponents as their definition has them, values within
  half of their step."""
  codes, exponents, width = rows.codes.cpu(), rows.exponents.cpu(), rows.width
  R, blocks = codes.shape[0], codes.shape[1] // 128
  pad = 128 * blocks - width
  assert not codes[:, width:].any(), "codes past the width"
  e = exponents.permute(1, 0, 2).flatten(1)
  assert (e[:, blocks:] == 1).all(), "exponents past the blocks"
  bad = ~torch.isfinite(torch.nn.functional.pad(y, (0, pad)).view(R, blocks, 128)).all(-1)
  assert torch.equal(e[:, :blocks] == 255, bad)
  y, off = (torch.nn.functional.pad(torch.where(torch.isfinite(y), t, 0.0), (0, pad)).view(R, blocks, 128) for t in (y, off))
  power = torch.ldexp(torch.ones(1, dtype=torch.float64), e[:, :blocks].long() - 127)
  top, slack = y.abs().amax(-1), off.amax(-1)
  fine = bad | (top - slack <= 464.0 * power) & ((e[:, :blocks] == 1) | (top + slack > 232.0 * power)) | (e[:, :blocks] == 246)
  assert fine.all(), "exponents"
  got = torch.nn.functional.pad(values(rows.codes, rows.exponents, width), (0, pad)).view(R, blocks, 128)
  m = y.abs() / power[..., None]
  step = torch.where(m < 2.0**-6, 2.0**-9, torch.exp2(torch.floor(torch.log2(m.clamp(min=2.0**-6))) - 3)).clamp(max=32.0)
  most = 0.5 * step * power[..., None] + off * 1.0625        # (a value within `off` of the next binade has that one's step: an eighth more of it, halved)
  far = (got - y).abs() - most
  far[bad] = 0.0
  assert float(far.max()) <= 0, float(far.max())


def product(x, w, bias, residual, activation):
  """act(x w^T + residual + bias) of rows in 64 bits, what the activation is of, and how far fp32 may be off that:

  steps    of 2^-24, the sums of the magnitudes: at most one rounding a product
  groups   the sum over groups of eight neighbouring products of each group's largest magnitude"""
  y, size = x @ w.t(), x.abs() @ w.abs().t()
  for t in (residual, bias):
    if t is not None:
      y, size = y + t.double(), size + t.double().abs()
  groups = torch.zeros_like(y)
  for k in range(0, x.shape[1], 8):
    top = torch.zeros_like(y)
    for a, b in zip(x[:, k : k + 8].abs().unbind(1), w[:, k : k + 8].abs().unbind(1)):
      top = torch.maximum(top, a[:, None] * b[None, :])
    groups += top
  return (y * torch.sigmoid(y) if activation else y), y, (size, groups)


def product_off(y, before, sizes, depth, dtype, activation):
  """How far the kernels may be off act(...).  In fp32 every product is exact and a sum of `depth` has at most as many roundings and the two
  that follow.  For bf16 results the matrix instructions on codes cut each of eight neighbouring products to a grid of 2^-13 of the largest of
  them (toward zero; the largest itself is on it) before they add them in fp32: seven of those.  SiLU has a slope of at most 1.1 and six
  roundings, two of them of its exponent (|x| steps each)."""
  size, groups = sizes
  fp32 = dtype == torch.float32
  off = (depth + 2) * STEP * size + (0.0 if fp32 else 7 * 2.0**-13 * groups)
  if activation:
    off = 1.1 * off + (6 + 2 * before.abs()) * STEP * before.abs()
  return off + (STEP if fp32 else 2.0**-8) * (y.abs() + off)
