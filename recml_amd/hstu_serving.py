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
  ids        int64 [batch, max_len], the events' items, where there are timestamps and more than one block; or None

  An event's time bias reads the next event's time, and the blocks above the first keep keys and values of what the attention gave the
  event.  So with timestamps those of a user's last event stand until the next one comes, and are made again then: a step runs, and
  writes, the last kept event too.

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
    self._items = torch.zeros_like(self._times) if timestamps and len(blocks) > 1 else None
    self.ids = None if self._items is None else self._items[:-1].view(batch, max_len)

  @property
  def batch(self) -> int:
    return self.lengths.shape[0]

  def reset(self, users=None) -> None:
    """Forgets the histories of `users` (an index, a mask or a slice; all by default)."""
    self.lengths[slice(None) if users is None else users] = 0

  def _note(self, ids, timestamps, users, places):
    """Keeps the times of new events, and their items where they are asked for again (all shaped alike); places past max_len are not kept."""
    if (self.timestamps is None) != (timestamps is None):
      raise ValueError("a cache made with timestamps=True takes `timestamps` with every event, and no other cache does")
    if timestamps is not None:
      if timestamps.shape != places.shape:
        raise ValueError(f"timestamps must be {tuple(places.shape)}, got {tuple(timestamps.shape)}")
      at = torch.where(places < self.max_len, users * self.max_len + places, self._times.numel() - 1).reshape(-1)
      self._times[at] = timestamps.to(torch.int64).reshape(-1)
      if self._items is not None:
        self._items[at] = ids.to(torch.int64).reshape(-1)

  def _with_last(self, ids, places, starts, lengths, offsets, max_new):
    """New events with each user's last kept one in front of them: (ids, places, starts, offsets, max_new, rows), laid out like the new events
    alone, `rows` where those are among them (packed; padded ones are all but each user's first).  A user without a kept event has a row
    at place -1 there, which joins nothing; one without a new event, or past max_len, gets `starts` under which none of its rows does."""
    at, full = starts.to(torch.int64) - 1, starts >= self.max_len
    last = self.ids.gather(1, at.clamp(0, self.max_len - 1)[:, None])
    ids = ids.to(torch.int64)
    if offsets is None:
      rows, most = None, ids.shape[1] + 1
      ids, places = torch.cat([last, ids], 1), torch.cat([at[:, None], places], 1)
    else:
      T, B = ids.shape[0], self.batch
      ends = offsets.to(torch.int64).clamp(0, T)
      firsts = ends[:-1] + torch.arange(B, device=ids.device)
      rows = torch.arange(T, device=ids.device)
      rows = rows + torch.searchsorted(ends[:-1], rows, right=True)
      together = torch.zeros((2, T + B), dtype=torch.int64, device=ids.device)
      together[:, rows] = torch.stack([ids, places.to(torch.int64)])
      together[:, firsts] = torch.stack([last[:, 0], at])
      ids, places = together
      offsets, most = (ends + torch.arange(B + 1, device=ids.device)).to(torch.int32), min(int(max_new), T) + 1
      max_new, full = most, full | (lengths == starts)
    starts = torch.where(full, -1 - most, starts - 1)
    return ids, places, starts, offsets, max_new, rows
