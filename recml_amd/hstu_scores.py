"""Log probabilities of given tokens from logits (libhstu_serve.so): torch tensors in, HIP kernels behind the C ABI.

  token_log_probs    log probabilities, the rows' entropy, the largest alternatives; differentiable

What a model's head leaves to be done (recml/layers/keras/hstu.py:617-621): a training loss over its logits, the scores of
candidate items, and the items to recommend.  One pass over the logits forward, one each way backward, sums in fp32; on a GPU
only; there is no other implementation behind this name.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from recml_amd import _lib_serve
from recml_amd import _native
from recml_amd.hstu_cache_ops import _DTYPES, _call, _check_gpu

MAX_TOP = 256
MAX_VOCAB = 1 << 30


class TokenLogProbs(NamedTuple):
  """What token_log_probs returns; what was not asked for is None."""

  log_probs: Optional[torch.Tensor]
  entropy: Optional[torch.Tensor]
  top_log_probs: Optional[torch.Tensor]
  top_tokens: Optional[torch.Tensor]


def _args(x, tokens, top):
  a = _lib_serve.HstuLogProbsArgs()
  a.struct_size, a.version = C.sizeof(a), _lib_serve.ABI_VERSION
  a.logits, a.rows, a.stride, a.vocab, a.dtype = x.data_ptr(), x.shape[0], x.stride(0) if x.shape[0] > 1 else 0, x.shape[1], _DTYPES[x.dtype]
  a.count, a.top = (tokens.shape[1] if tokens is not None else 0), top
  a.tokens = None if tokens is None else tokens.data_ptr()
  return a


def _forward(x, tokens, top, entropy, stats):
  """x [R, V], tokens [R, C] or None -> fp32 log_probs [R, C], entropy [R], stats [R, 3], top_log_probs [R, top], top_tokens."""
  new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=x.device)
  R = x.shape[0]
  lp = None if tokens is None else new(*tokens.shape)
  ent = new(R) if entropy else None
  st = new(R, 3) if stats else None
  tl, ti = (new(R, top), new(R, top, dtype=torch.int64)) if top else (None, None)
  a = _args(x, tokens, top)
  for name, t in (("log_probs", lp), ("entropy", ent), ("stats", st), ("top_log_probs", tl), ("top_tokens", ti)):
    if t is not None:
      setattr(a, name, t.data_ptr())
  need = _lib_serve.load().hstu_log_probs_workspace_bytes(C.byref(a))
  if need:
    ws = new(need, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
  _call("hstu_log_probs_fwd", a, x.device)
  return lp, ent, st, tl, ti


class _TokenLogProbsFn(torch.autograd.Function):
  """token_log_probs with the gradient of the logits through the HIP kernel."""

  @staticmethod
  def forward(ctx, x, tokens, top, entropy):
    lp, ent, st, tl, ti = _forward(x, tokens, top, entropy, True)
    ctx.top = top
    ctx.save_for_backward(x, tokens, st, ti)
    if ti is not None:
      ctx.mark_non_differentiable(ti)
    ctx.set_materialize_grads(False)
    return lp, ent, tl, ti

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, g_lp, g_ent, g_top, _):
    x, tokens, st, ti = ctx.saved_tensors
    if g_lp is None and g_ent is None and g_top is None:
      return None, None, None, None
    d = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _args(x, tokens, ctx.top)
    a.stats, a.d_logits, a.d_stride = st.data_ptr(), d.data_ptr(), d.stride(0)
    a.top_tokens = None if ti is None else ti.data_ptr()
    keep = [None if g is None else g.to(torch.float32).contiguous() for g in (g_lp, g_ent, g_top)]
    for name, g in zip(("g_tokens", "g_entropy", "g_top"), keep):
      if g is not None:
        setattr(a, name, g.data_ptr())
    _call("hstu_log_probs_bwd", a, x.device)
    del keep
    return d, None, None, None


def token_log_probs(logits, tokens=None, *, top: int = 0, entropy: bool = False) -> TokenLogProbs:
  """Log probabilities of `tokens` under softmax(logits), and what else is asked for, in fp32.

  Args:
    logits: [..., V], float32 or bfloat16 (a copy is made where the last axis is not contiguous or the others do not flatten to
      one row stride).
    tokens: integers [...] (one token a row) or [..., C] (C of them), or None.  A negative token asks for nothing: 0, and no
      gradient.  A token past the vocabulary gives NaN.
    top: how many of the row's largest log probabilities to return with their tokens (up to 256 and V), in falling order, ties by
      the lower token.
    entropy: whether to return the rows' entropy, -sum p log p.

  Entries of -inf are tokens that cannot occur.  A row with a NaN, with +inf, or with nothing but -inf is NaN throughout.
  Differentiable in the logits, through log_probs, entropy and top_log_probs.  Captured into a graph with a gradient, it raises where an
  eager graph of the same leaves lives: their accumulators are not the captured stream's, and the backward pass would end the process."""
  got = _native.token_log_probs(logits, tokens, top, entropy)
  if got is not None:
    return TokenLogProbs(*got)
  _check_gpu("logits", logits)
  if logits.dtype not in _DTYPES:
    raise ValueError(f"logits: unsupported dtype {logits.dtype}: use float32 or bfloat16")
  if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
    raise ValueError(f"logits must be [..., V] with V from 1 to {MAX_VOCAB}, got {tuple(logits.shape)}")
  lead, V = tuple(logits.shape[:-1]), logits.shape[-1]
  top = int(top)
  if not 0 <= top <= min(MAX_TOP, V):
    raise ValueError(f"top must lie between 0 and {min(MAX_TOP, V)}, got {top}")
  ids = None
  if tokens is not None:
    _check_gpu("tokens", tokens)
    if tokens.dtype.is_floating_point or tokens.dtype == torch.bool or tokens.device != logits.device:
      raise ValueError(f"tokens must hold integers on {logits.device}, got {tokens.dtype} on {tokens.device}")
    shape = tuple(tokens.shape)
    if shape != lead and not (len(shape) == len(lead) + 1 and shape[:-1] == lead):
      raise ValueError(f"tokens must be {lead} or {lead + ('C',)}, got {shape}")
    if shape != lead and shape[-1] > MAX_VOCAB:
      raise ValueError(f"at most {MAX_VOCAB} tokens a row, got {shape}")
    if tokens.numel():
      ids = tokens.to(torch.int64).reshape(-1, 1 if shape == lead else shape[-1]).contiguous()
  elif not top and not entropy:
    raise ValueError("nothing is asked for: pass tokens, top or entropy=True")
  x = logits if logits.dim() == 2 else logits.reshape(-1, V)
  if x.stride(1) != 1 and V > 1:
    x = x.contiguous()
  if (torch.is_grad_enabled() and logits.requires_grad) or _native.has_tangent(logits):
    lp, ent, tl, ti = _TokenLogProbsFn.apply(x, ids, top, bool(entropy))
  else:
    lp, ent, _, tl, ti = _forward(x, ids, top, bool(entropy), False)
  if tokens is not None:
    lp = torch.empty(tokens.shape, dtype=torch.float32, device=logits.device) if lp is None else lp.reshape(tokens.shape)
  return TokenLogProbs(lp, None if ent is None else ent.reshape(lead), None if tl is None else tl.reshape(*lead, top),
                       None if ti is None else ti.reshape(*lead, top))
