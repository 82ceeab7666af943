"""The paged key/value cache of the attention half.

One pool ``pages [n_pages, layers, 2, kv_heads, page_size, head_dim]`` (a page holds its
tokens' keys and values of all layers in one contiguous block, so copying a page is one
copy) and its bookkeeping, all on the device: ``refs [n_pages]`` (sequences that hold a
page; 0: free), ``tables [max_seqs, max_pages]`` (-1: no page) and ``lens [max_seqs]``.
The reference keeps one slot of fixed length per sequence instead
(engine/runtime/kv_cache.py:220).

Only the calls change these.  Lengths only grow: tokens are taken back (rejected drafts) by
``fork`` of those that stay into an empty slot and ``free`` of the old one; a length lowered by
hand would lose the pages behind it and let new tokens into pages that branches share.

The calls run in stream order without a host sync and can be captured in CUDA graphs when
their lists are device tensors.  ``grow`` and ``fork`` return ``ok`` (int32, one per
request; 0: refused, nothing changed) on the device.
"""
from __future__ import annotations

import torch

from . import ops


class PagedKVCache:
    def __init__(self, n_pages: int, page_size: int, layers: int, kv_heads: int, head_dim: int,
                 max_seqs: int, max_len: int, device="cuda"):
        if min(n_pages, page_size, layers, kv_heads, head_dim, max_seqs, max_len) < 1:
            raise ValueError("PagedKVCache: sizes must be positive")
        if page_size not in (16, 32, 64, 128):
            raise ValueError("PagedKVCache: page_size must be 16, 32, 64 or 128")
        if head_dim not in (64, 128, 256):
            raise ValueError("PagedKVCache: head_dim must be 64, 128 or 256")
        i32 = dict(dtype=torch.int32, device=device)
        self.pages = torch.zeros((n_pages, layers, 2, kv_heads, page_size, head_dim),
                                 dtype=torch.bfloat16, device=device)
        self.refs = torch.zeros(n_pages, **i32)
        self.tables = torch.full((max_seqs, -(-max_len // page_size)), -1, **i32)
        self.lens = torch.zeros(max_seqs, **i32)

    @property
    def page_size(self) -> int:
        return self.pages.shape[-2]

    def k(self, layer: int) -> torch.Tensor:
        """Layer's keys [n_pages, kv_heads, page_size, head_dim] (a view)."""
        return self.pages[:, layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        """Layer's values [n_pages, kv_heads, page_size, head_dim] (a view)."""
        return self.pages[:, layer, 1]

    def _list(self, x) -> torch.Tensor:
        return torch.as_tensor(x, dtype=torch.int32, device=self.refs.device)

    def grow(self, slots, add) -> torch.Tensor:
        """Room for ``add[i]`` more tokens of sequence ``slots[i]``."""
        return ops.pages_grow(self.refs, self.tables, self.lens, self._list(slots),
                              self._list(add), self.page_size)

    def fork(self, src, dst, keep=None) -> torch.Tensor:
        """Empty sequences ``dst`` become the first ``keep`` tokens (default: all) of ``src``.  Refused
        (ok 0) among others where ``keep`` ends inside a page that ``src`` has given up behind a
        window."""
        src = self._list(src)
        if keep is None:   # (the call itself refuses sources out of range)
            keep = self.lens[src.clamp(0, self.lens.shape[0] - 1)]
        keep = self._list(keep)
        return ops.pages_fork(self.pages, self.refs, self.tables, self.lens, src,
                              self._list(dst), keep)

    def free(self, slots, window: int = 0, sinks: int = 0) -> None:
        """Give up the sequences' pages; with a window, only those it no longer sees."""
        ops.pages_free(self.refs, self.tables, self.lens, self._list(slots), self.page_size,
                       window, sinks)

    def compact(self):
        """Move the live pages to the front; returns (live [1], remap [n_pages])."""
        return ops.pages_compact(self.pages, self.refs, self.tables)
