"""The operators of a block's steps on rows kept in 8 bits, as timed cases.

A case's `kind` says what it calls:

  norm     recml_amd.norm_rows8 or quantize_rows, and Rows8.values: rows normed (layer norm or root mean square; other rows added first,
           multiplied by a gate after) and quantised, and what the codes stand for
  product  recml_amd.gemm_rows8: rows in 8 bits times a weight in 8 bits, with what a block puts behind the product
  steps    a block's steps around its attention as one run: norm, projections, norm and gate, output product with the residual

Rows in 8 bits are e4m3 codes [rows, 128 blocks] (uint8, zeros past the width) whose blocks of 128 values share a power of two: exponents
[ceil(blocks / 4), rows, 4] (uint8, biased by 127).  The power is the smallest under which the block's largest magnitude rounds to a code.
A weight is kept by the same rule as rows along the contraction, one for each of its output columns.

Sizes are those of recml_amd.workloads, bench.py and the example model; `draw` spreads the same kinds over their range.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "bf16": 2}
_EPS = 1e-6


def _norm(name, rows, width, *, norm="layer", add=False, gate=False, dtype="bf16"):
  return dict(name=name, kind="norm", rows=rows, width=width, norm=norm, add=add, gate=gate, dtype=dtype)


def _product(name, rows, depth, cols, *, act=False, bias=False, residual=False, dtype="bf16"):
  return dict(name=name, kind="product", rows=rows, depth=depth, cols=cols, act=act, bias=bias, residual=residual, dtype=dtype)


def _steps(name, rows, width, *, dtype="bf16"):
  return dict(name=name, kind="steps", rows=rows, width=width, dtype=dtype)


def listed():
  return [
      # one user's next event in front of the projections: nothing but latency counts
      _norm("norm of one event", 1, 512),
      # the headline batch's packed tokens, the attention's norm with the U gate
      _norm("norm and gate, jagged batch", 16398, 1024, gate=True),
      # the ranking model's whole batch, the residual added on the way: the largest
      _norm("residual and rms norm", 131072, 512, norm="rms", add=True),
      # Keras' default type, an odd width
      _norm("odd width, fp32", 4097, 1001, add=True, dtype="fp32"),
      # a million items' embeddings (or a table's rows) taken into 8 bits, once
      _norm("embeddings quantised", 1000000, 64, norm="none"),
      # one user's next event through the projections of the headline model
      _product("projection of one event", 1, 1024, 4096, act=True),
      # an event of each user over the whole vocabulary: the head's logits
      _product("logits of 64 events", 64, 512, 1000000),
      # the ranking model's projections over a packed batch
      _product("projections, ranking batch", 73728, 512, 2048, act=True),
      # odd sizes throughout, Keras' default type
      _product("odd sizes, fp32", 1237, 1001, 777, bias=True, residual=True, dtype="fp32"),
      # a product large enough to run at the matrix cores' rate
      _product("large product", 16384, 8192, 8192),
      # a serving step of the headline model: every user's next event through a block's steps
      _steps("a block's steps, 64 events", 64, 1024),
      # and its jagged batch
      _steps("a block's steps, jagged batch", 16398, 1024),
  ]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
  """One more case of the listed kinds, that costs no more than the largest listed one of its kind."""
  while True:
    kind = rng.choice(("norm", "norm", "product", "product", "product", "steps"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    if kind == "norm":
      norm = rng.choice(("layer", "layer", "rms", "none"))
      plain = norm == "none"
      case = _norm("", _log_int(rng, 1, 1000000), _log_int(rng, 8, 8192), norm=norm, add=not plain and rng.random() < 0.4,
                   gate=not plain and rng.random() < 0.3, dtype=dtype)
      cap = "residual and rms norm"
    elif kind == "product":
      act = rng.random() < 0.4
      case = _product("", _log_int(rng, 1, 131072), _log_int(rng, 8, 8192), _log_int(rng, 8, 200000), act=act, bias=rng.random() < 0.4,
                      residual=not act and rng.random() < 0.4, dtype=dtype)
      cap = "large product"
    else:
      case = _steps("", _log_int(rng, 1, 32768), 8 * _log_int(rng, 2, 256), dtype=dtype)
      cap = "large product"
    del case["name"]
    most, cost = work(next(c for c in listed() if c["name"] == cap)), work(case)
    if cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]:
      return case


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------


def _row_bytes(width):
  """Codes of a row with its exponents."""
  return width + -(-width // 128)


def _norm_bytes(rows, width, elem, add, gate):
  return rows * (width * elem * (1 + 2 * add + gate) + _row_bytes(width))


def _product_bytes(rows, depth, cols, elem, residual):
  return (rows + cols) * _row_bytes(depth) + rows * cols * elem * (1 + residual)


def work(case):
  e, R = _BYTES[case["dtype"]], case["rows"]
  if case["kind"] == "norm":
    # (the values are read back in bf16)
    return {"bytes": _norm_bytes(R, case["width"], e, case["add"], case["gate"]) + R * (_row_bytes(case["width"]) + 2 * case["width"]),
            "flops": 12 * R * case["width"]}
  if case["kind"] == "product":
    return {"bytes": _product_bytes(R, case["depth"], case["cols"], e, case["residual"]), "flops": 2 * R * case["depth"] * case["cols"]}
  W = case["width"]
  return {"bytes": R * W * e * (1 + 4 + 3 + 1) + 5 * W * _row_bytes(W), "flops": 10 * R * W * W}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


class _Draws:
  """Device-side random values of one seed."""

  def __init__(self, seed):
    self.dev = torch.device("cuda")
    self.gen = torch.Generator(device=self.dev).manual_seed(seed)

  def normal(self, shape, std, dtype=torch.float32, mean=0.0):
    return torch.randn(shape, device=self.dev, generator=self.gen).mul_(std).add_(mean).to(dtype)


def _activations(r, rows, width, dtype):
  """Rows whose channels differ in size, as a residual stream's do: most near 1, some in a hundred several times that."""
  spread = torch.exp(0.5 * r.normal((width,), 1.0)) * torch.where(r.normal((width,), 1.0) > 2.3, 8.0, 1.0)
  return r.normal((rows, width), 1.0).mul_(spread).to(dtype)


def prepare(case, seed):
  r = _Draws(seed)
  dt, R = _DTYPES[case["dtype"]], case["rows"]
  state = dict(case, dtype=dt)
  if case["kind"] == "norm":
    W = case["width"]
    state["x"] = _activations(r, R, W, dt)
    state["gamma"], state["beta"] = r.normal((W,), 0.2, dt, 1.0), r.normal((W,), 0.1, dt)
    state["other"] = _activations(r, R, W, dt) if case["add"] else None
    state["u"] = r.normal((R, W), 0.5, dt) if case["gate"] else None
    return state
  if case["kind"] == "product":
    K, N = case["depth"], case["cols"]
    state["x"] = _quantised(_activations(r, R, K, torch.float32))
    state["w"] = _quantised(r.normal((N, K), K ** -0.5))
    state["b"] = r.normal((N,), 0.1, dt) if case["bias"] else None
    state["c"] = r.normal((R, N), 1.0, dt) if case["residual"] else None
    return state
  W = case["width"]
  state["x"], state["attn"] = _activations(r, R, W, dt), r.normal((R, W), 0.1, dt)
  state["w"], state["w_out"] = _quantised(r.normal((4 * W, W), W ** -0.5)), _quantised(r.normal((W, W), W ** -0.5))
  for name in ("in", "attn"):
    state[name + "_gamma"], state[name + "_beta"] = r.normal((W,), 0.2, dt, 1.0), r.normal((W,), 0.1, dt)
  return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _power(e):
  """2^e in fp32 for whole e in [-126, 127], by its bits: a device's pow is not exact."""
  return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
  """fp32 rows [R, W] as codes [R, 128 blocks] and exponents [ceil(blocks / 4), R, 4].  Every step is exact: the powers of two scale
  without rounding, so the borders between codes are where the definition has them."""
  R, W = x.shape
  blocks = -(-W // 128)
  groups = -(-blocks // 4)
  x = torch.nn.functional.pad(x, (0, 128 * blocks - W)).view(R, blocks, 128)
  top = x.abs().amax(-1)
  mantissa, exponent = torch.frexp(top)
  e = exponent - 9 + (mantissa > 0.90625).to(exponent.dtype)
  e = torch.where(top > 0, e, -126).clamp(-126, 119)                     # (no code stands for more than fp32 holds)
  y = (x * _power(-e)[..., None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).view(R, 128 * blocks)
  kept = torch.ones((R, 4 * groups), dtype=torch.uint8, device=x.device)
  kept[:, :blocks] = (e + 127).to(torch.uint8)
  return y, kept.view(R, groups, 4).transpose(0, 1).contiguous()


def _values(codes, exponents, width):
  """fp32 rows [R, width] of codes and exponents."""
  R, blocks = codes.shape[0], codes.shape[1] // 128
  e = exponents.transpose(0, 1).reshape(R, -1)[:, :blocks].to(torch.int32) - 127
  return (codes.view(torch.float8_e4m3fn).float().view(R, blocks, 128) * _power(e)[..., None]).view(R, -1)[:, :width]


def _normed(x, gamma, beta, kind):
  """Rows of fp32 normed over their last axis."""
  if kind == "layer":
    x = x - x.mean(-1, keepdim=True)
  y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * gamma.float()
  return y if beta is None else y + beta.float()


def _silu(x):
  return x / (1 + torch.exp(-x))


def _norm_plain(s):
  x, out = s["x"].float(), {}
  if s["other"] is not None:
    out["sum"] = (x + s["other"].float()).to(s["dtype"])
    x = out["sum"].float()
  if s["norm"] != "none":
    x = _normed(x, s["gamma"], s["beta"] if s["norm"] == "layer" else None, s["norm"])
  if s["u"] is not None:
    x = x * s["u"].float()
  out["values"] = _values(*_quantised(x), s["width"]).to(torch.bfloat16)
  return out


def _product_plain(s):
  y = _values(*s["x"], s["depth"]) @ _values(*s["w"], s["depth"]).t()
  if s["c"] is not None:
    y = y + s["c"].float()
  if s["b"] is not None:
    y = y + s["b"].float()
  return (_silu(y) if s["act"] else y).to(s["dtype"])


def _steps_plain(s):
  W, x = s["width"], s["x"].float()
  normed = _values(*_quantised(_normed(x, s["in_gamma"], s["in_beta"], "layer")), W)
  uqkv = _silu(normed @ _values(*s["w"], W).t()).to(s["dtype"])
  gated = _normed(s["attn"].float(), s["attn_gamma"], s["attn_beta"], "layer") * uqkv[:, :W].float()
  out = _values(*_quantised(gated), W) @ _values(*s["w_out"], W).t() + x
  return {"uqkv": uqkv, "out": out.to(s["dtype"])}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _own_run(s):
  import recml_amd
  if s["kind"] == "norm":
    if s["norm"] == "none":
      return {"values": recml_amd.quantize_rows(s["x"]).values()}
    layer = s["norm"] == "layer"
    got = recml_amd.norm_rows8(s["x"], s["gamma"], s["beta"] if layer else None, _EPS, gate=s["u"], add=s["other"], rms=not layer)
    return {"values": got.values()} if s["other"] is None else {"sum": got[1], "values": got[0].values()}
  W = s["depth"] if s["kind"] == "product" else s["width"]
  w = recml_amd.Rows8(*s["w"], W)
  if s["kind"] == "product":
    return recml_amd.gemm_rows8(recml_amd.Rows8(*s["x"], W), w, s["b"], s["act"], residual=s["c"], dtype=s["dtype"])
  rows = recml_amd.norm_rows8(s["x"], s["in_gamma"], s["in_beta"], _EPS)
  uqkv = recml_amd.gemm_rows8(rows, w, None, True, dtype=s["dtype"])
  gated = recml_amd.norm_rows8(s["attn"], s["attn_gamma"], s["attn_beta"], _EPS, gate=uqkv[:, :W])
  return {"uqkv": uqkv, "out": recml_amd.gemm_rows8(gated, recml_amd.Rows8(*s["w_out"], W), residual=s["x"], dtype=s["dtype"])}


def run(state):
  if own:
    return _own_run(state)
  return {"norm": _norm_plain, "product": _product_plain, "steps": _steps_plain}[state["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_power(e):
  """2^e in 64 bits for whole e."""
  return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_levels(dev):
  """The magnitudes of the codes in rising order (the last code is no number)."""
  e4m3 = [f / 512 for f in range(8)] + [(1 + f / 8) * 2.0 ** (e - 7) for e in range(1, 16) for f in range(8)]
  return torch.tensor(e4m3[:127], dtype=torch.float64, device=dev)


def _exact_stored(x):
  """What rows become in 8 bits: the nearest level (ties to the even code) times the block's power."""
  levels = _exact_levels(x.device)
  most = levels[-1] + 16.0                                 # half a step past the largest code rounds to it
  parts = []
  for block in x.split(128, -1):
    top = block.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / most)).clamp(-200, 200)
    e = torch.where(top > most * _exact_power(e), e + 1, torch.where(top <= most * _exact_power(e - 1), e - 1, e)).clamp(-126, 119)
    power = torch.where(top > 0, _exact_power(e), 1.0)
    m = block.abs() / power
    hi = torch.searchsorted(levels, m.contiguous()).clamp(1, len(levels) - 1)
    lo = hi - 1
    below, above = m - levels[lo], levels[hi] - m
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    parts.append(levels[code] * power * torch.sign(block))
  return torch.cat(parts, -1)


def _exact_values(codes, exponents, width, rows=slice(None)):
  """Kept rows in 64 bits."""
  c = codes[rows].long()
  e = exponents[:, rows].permute(1, 0, 2).flatten(1)[:, : c.shape[1] // 128]
  y = _exact_levels(c.device)[(c % 128).clamp(max=126)] * _exact_power(e.double() - 127.0).repeat_interleave(128, -1)
  return torch.where(c >= 128, -y, y)[:, :width]


def _exact_normed(x, gamma, beta, layer):
  x = x.double()
  mean = x.mean(-1, keepdim=True) if layer else 0.0
  y = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + _EPS) * gamma.double()
  return y if beta is None else y + beta.double()


def _exact_silu(x):
  return x * torch.sigmoid(x)


def exact(case, seed):
  s = prepare(case, seed)
  R, W = case["rows"], case["depth"] if case["kind"] == "product" else case["width"]
  w = None if case["kind"] == "norm" else _exact_values(*s["w"], W).t().contiguous()
  w_out = _exact_values(*s["w_out"], W).t().contiguous() if case["kind"] == "steps" else None
  parts, step = [], max(1, (1 << 25) // (W + 2 * (0 if w is None else w.shape[1])))
  for r in range(0, R, step):
    at, out = slice(r, r + step), {}
    if case["kind"] == "norm":
      x = s["x"][at].double()
      if s["other"] is not None:
        out["sum"] = x + s["other"][at].double()
        x = out["sum"].to(s["dtype"])                      # (the norm is of the rows that are handed on)
      if s["norm"] != "none":
        x = _exact_normed(x, s["gamma"], s["beta"] if s["norm"] == "layer" else None, s["norm"] == "layer")
      out["values"] = _exact_stored(x.double() if s["u"] is None else x * s["u"][at].double())
    elif case["kind"] == "product":
      y = _exact_values(*s["x"], W, at) @ w
      y = y if s["c"] is None else y + s["c"][at].double()
      y = y if s["b"] is None else y + s["b"].double()
      out["out"] = _exact_silu(y) if s["act"] else y
    else:
      y = _exact_silu(_exact_stored(_exact_normed(s["x"][at], s["in_gamma"], s["in_beta"], True)) @ w)
      u = y[:, :W].to(s["dtype"]).double()                 # (the gate is of the rows that are handed on)
      gated = _exact_stored(_exact_normed(s["attn"][at], s["attn_gamma"], s["attn_beta"], True) * u)
      out = {"uqkv": y, "out": gated @ w_out + s["x"][at].double()}
    parts.append(out)
  got = {name: torch.cat([part[name] for part in parts]) for name in parts[0]}
  return got["out"] if case["kind"] == "product" else got
