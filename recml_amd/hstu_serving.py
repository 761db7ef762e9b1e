"""What an HSTU model keeps of its users' histories between calls (HSTU.prefill and HSTU.extend fill and read it)."""

from __future__ import annotations

import torch

from recml_amd import hstu_cache_ops


class HSTUCache:
  """The kept histories of `batch` users: every layer's keys and values in 4 or 8 bits, how many events each user has, and, where
  the model's attention has a timestamp bias, when they were.

  layers     one KVPages per block; they share `page_table` [batch, n]
  lengths    int32 [batch] on the GPU
  timestamps int64 [batch, max_len], or None

  By default every user owns the pages for `max_len` events.  With `pages` and a `page_table` of the caller's (int32, -1 where a user
  has no page) a pool is shared out as the caller likes; events without a page are dropped and attended to by nobody.  `max_len`
  is the length that the model's full call would have: the normaliser and the position table's extent."""

  def __init__(self, blocks, batch: int, max_len: int, *, bits: int = 4, page_size: int = 64, pages: int | None = None, page_table=None,
               timestamps: bool = False, device=None):
    blocks = list(blocks)
    if batch < 1 or max_len < 1:
      raise ValueError(f"batch and max_len must be positive, got {batch} and {max_len}")
    if (pages is None) != (page_table is None):
      raise ValueError("`pages` and `page_table` go together")
    each = -(-max_len // page_size)
    if page_table is None:
      pages = batch * each
      page_table = torch.arange(pages, dtype=torch.int32, device=device).reshape(batch, each)
    elif page_table.dim() != 2 or page_table.shape[0] != batch:
      raise ValueError(f"page_table must be [{batch}, n], got {tuple(page_table.shape)}")
    self.max_len = int(max_len)
    self.page_table = page_table
    self.layers = [hstu_cache_ops.KVPages.empty(pages, page_size, b.num_heads, b.head_dim, bits=bits, device=device) for b in blocks]
    self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
    # (one entry more than there are places, for the times of events that have none)
    self._times = torch.zeros(batch * max_len + 1, dtype=torch.int64, device=device) if timestamps else None
    self.timestamps = self._times[:-1].view(batch, max_len) if timestamps else None

  @property
  def batch(self) -> int:
    return self.lengths.shape[0]

  def reset(self, users=None) -> None:
    """Forgets the histories of `users` (an index, a mask or a slice; all by default)."""
    self.lengths[slice(None) if users is None else users] = 0

  def _note_times(self, timestamps, users, places):
    """Keeps the times of new events (all shaped alike); places past max_len are not kept."""
    if (self.timestamps is None) != (timestamps is None):
      raise ValueError("a cache made with timestamps=True takes `timestamps` with every event, and no other cache does")
    if timestamps is not None:
      if timestamps.shape != places.shape:
        raise ValueError(f"timestamps must be {tuple(places.shape)}, got {tuple(timestamps.shape)}")
      at = torch.where(places < self.max_len, users * self.max_len + places, self._times.numel() - 1)
      self._times[at.reshape(-1)] = timestamps.to(torch.int64).reshape(-1)
