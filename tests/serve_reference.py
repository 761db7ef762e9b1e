"""The serving operators in 64 bits, element by element from their definitions (CPU tensors in, CPU tensors out)."""

import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [f / 512 for f in range(8)] + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8)][:119]


def stored(x, bits):
  """What rows [..., d] become in the cache."""
  levels = torch.tensor(E2M1 if bits == 4 else E4M3, dtype=torch.float64)
  most = 7.0 if bits == 4 else 464.0
  rows = x.double().reshape(-1, x.shape[-1])
  out = torch.empty_like(rows)
  for r, row in enumerate(rows):
    if not torch.isfinite(row).all():
      out[r] = math.nan
      continue
    for c in range(0, len(row), 32):
      block = row[c : c + 32]
      e, top = -126, float(block.abs().max())
      if top > 0:
        e = max(-126, math.frexp(top)[1] - 20)
        while top > most * 2.0**e:
          e += 1
      e = min(e, 125 if bits == 4 else 119)
      m = block.abs() / 2.0**e
      off = (m[:, None] - levels[None, :]).abs()
      near = off == off.min(1, keepdim=True).values
      code = torch.where(near[:, 0::2].any(1), 2 * near[:, 0::2].int().argmax(1), 2 * near[:, 1::2].int().argmax(1) + 1)
      out[r, c : c + 32] = torch.copysign(levels[code] * 2.0**e, block)
  return out.reshape(x.shape)


def values(codes, scales, bits, d):
  """What codes [pages, H, size, bytes] and exponents [pages, H, blocks, size] stand for: [pages, H, size, d]."""
  levels = torch.tensor(E2M1 if bits == 4 else E4M3 + [math.nan], dtype=torch.float64)
  c = codes.long()
  if bits == 4:
    c = torch.stack([c % 16, c // 16], -1).flatten(-2)
    y = levels[c % 8] * (1.0 - 2.0 * (c // 8))
  else:
    y = levels[c % 128] * (1.0 - 2.0 * (c // 128))
  e = scales.long().transpose(-1, -2)
  power = torch.where(e == 255, math.nan, torch.ldexp(torch.ones(1, dtype=torch.float64), e - 127))
  return y * power.repeat_interleave(32, -1)[..., :d]


def bucket(gap, size=0.301):
  x = gap.abs().clamp(1, 10**9).to(torch.float32).double()
  return torch.floor(torch.log(x) / float(torch.tensor(size, dtype=torch.float32))).long()


def attention(q, k, v, *, length, max_len, held, n=None, alpha=1.0, pos_bias=None, timestamps=None, ts_bias=None, ts_bucket_size=0.301):
  """One sequence: q [m, H, d], k and v [places, H, d] (64 bits), `held` [places] whether the cache holds the place.
  Returns the rows, and how far fp32 sums and logits may be off and what the weights' rounding is relative to."""
  m, H, d = q.shape
  q = q.double()
  i = torch.arange(length - m, length)
  limit = min(length, max_len, k.shape[0])
  j = torch.arange(limit)
  keep = (j[None, :] <= i[:, None]) & held[None, :limit] & (i[:, None] >= 0) & (i[:, None] < limit)
  # (masked places may hold anything)
  seen = keep.any(0)
  k = torch.where(seen[:, None, None], k[:limit], 0.0)
  v = torch.where(seen[:, None, None], v[:limit], 0.0)
  x = alpha * torch.einsum("mhd,jhd->hmj", q, k)
  size = abs(alpha) * torch.einsum("mhd,jhd->hmj", q.abs(), k.abs())
  if pos_bias is not None:
    t = pos_bias.double().reshape(-1, 2 * max_len - 1)
    add = t[:, (max_len - 1 + j[None, :] - i[:, None]).clamp(0, 2 * max_len - 2)]
    x, size = x + add, size + add.abs()
  if ts_bias is not None:
    t = ts_bias.double().reshape(-1, ts_bias.shape[-1])
    nxt = torch.minimum(i + 1, torch.tensor(min(length, max_len) - 1)).clamp(min=0)
    b = bucket(timestamps[nxt][:, None] - timestamps[j][None, :], ts_bucket_size).clamp(max=t.shape[1] - 1)
    x, size = x + t[:, b], size + t[:, b].abs()
  w = torch.where(keep[None], x * torch.sigmoid(x), 0.0)
  n = max_len if n is None else n
  # logits: d + 4 roundings of at most 2^-24 of what is summed; silu: slope at most 1.1, a few last places of its own
  dw = torch.where(keep[None], 1.1 * (d + 4) * 2.0**-24 * size + 16 * 2.0**-24 * w.abs(), 0.0)
  kept = lambda a: torch.einsum("hmj,jhd->mhd", a, v.abs()) / n
  # NaN of a kept row stays in its pairs; 0 * NaN of the others is nothing
  out = torch.zeros((m, H, v.shape[-1]), dtype=torch.float64)
  for t in range(m):
    cols = keep[t].nonzero().flatten()
    out[t] = torch.einsum("hj,jhd->hd", w[:, t, cols], v[cols]) / n
  return out, kept(dw), kept(w.abs())


def attention_tolerance(out, logits_off, weights, length, dtype):
  """Elementwise: the logits' part, fp32 sums of `length` terms, and the roundings of the weights and of the result."""
  tol = logits_off + (length + 8) * 2.0**-24 * weights
  half = torch.finfo(dtype).eps / 2
  return tol + half * (weights if dtype == torch.bfloat16 else 2 * weights) * 1.01 + half * out.abs() + 1e-30


def log_probs(x, tokens, top, g_tokens=None, g_entropy=None, g_top=None):
  """Rows x [R, V] in 64 bits: (log_probs, entropy, top_log_probs, top_tokens, d_logits), and the log-probabilities of all."""
  x = x.double()
  lp = torch.log_softmax(x, -1)
  p = lp.exp()
  bad = torch.isnan(lp).any(-1, keepdim=True)
  plogp = torch.where(p > 0, p * lp, 0.0)
  h = torch.where(bad[:, 0], math.nan, -plogp.sum(-1))
  ask = tokens.clamp(0, x.shape[1] - 1)
  picked = torch.where(tokens < 0, 0.0, torch.where(tokens >= x.shape[1], math.nan, lp.gather(1, ask)))
  order = torch.where(torch.isnan(x), math.inf, x)
  first = torch.sort(torch.where(torch.isnan(x), 1, 0), dim=-1, descending=True, stable=True).indices
  first = first.gather(1, torch.sort(order.gather(1, first), dim=-1, descending=True, stable=True).indices)[:, :top]
  g = torch.zeros_like(x)
  total = torch.zeros((x.shape[0], 1), dtype=torch.float64)
  if g_tokens is not None:
    gt = torch.where(tokens < 0, 0.0, torch.where(tokens >= x.shape[1], math.nan, g_tokens.double()))
    total = total + gt.sum(-1, keepdim=True)
    g = g.scatter_add(1, ask, gt)
  if g_top is not None:
    total = total + g_top.double().sum(-1, keepdim=True)
    g = g.scatter_add(1, first, g_top.double())
  inner = total.expand(x.shape)
  if g_entropy is not None:
    inner = inner + g_entropy.double()[:, None] * torch.where(p > 0, lp + h[:, None], 0.0)
  return picked, h, lp.gather(1, first), first, g - p * inner, lp, inner
