"""A paged key-value cache for rows of different lengths that may share pages.

``PagedKVCache`` holds the pools, the page table and the counts of one model's
cache and keeps them consistent through ``ops.paged_update``; all of it lives
on the device, so a step that forks, reserves and attends needs no host sync
and can be captured into a graph.  ``LoomDecoder.beam_search`` runs on it.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _lib, ops


class PagedKVCache:
    """Keys and values of ``layers`` layers for ``rows`` rows of up to ``max_len``
    tokens, in pages of ``page_size`` tokens (a power of two, 16 to 1024).

      k_pages, v_pages [layers, n_pages, kv_heads, page_size, head_dim]
      table [rows, max_pages] int32   pages of each row (-1: none)
      lens  [rows] int32              tokens each row holds (-1: no sequence)
      refs  [n_pages] int32           table entries that hold each page
      status [1] int32                pages that could not be had (see check)

    A row's last tokens are dropped by lowering its entry of lens.  n_pages defaults to what rows that share nothing need, which never runs out.
    """

    def __init__(self, layers: int, rows: int, max_len: int, kv_heads: int, head_dim: int, dtype: torch.dtype,
                 device="cuda", page_size: int = 64, n_pages: Optional[int] = None):
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if not 1 <= rows <= 1024:
            raise ValueError(f"rows must be 1 to 1024, got {rows}")
        self.page_size = int(page_size)
        max_pages = -(-int(max_len) // self.page_size)
        self.n_pages = rows * max_pages if n_pages is None else int(n_pages)
        if self.n_pages < 1:
            raise ValueError(f"n_pages must be at least 1, got {self.n_pages}")
        dev = torch.device(device)
        shape = (layers, self.n_pages, kv_heads, self.page_size, head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=dev)
        self.v_pages = torch.empty(shape, dtype=dtype, device=dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((rows, max_pages), -1, **i32)
        self.lens = torch.full((rows,), -1, **i32)
        self.refs = torch.zeros(self.n_pages, **i32)
        self.status = torch.zeros(1, **i32)
        self._used = torch.zeros(1, **i32)

    @property
    def rows(self) -> int:
        return self.table.shape[0]

    def reset(self) -> None:
        """Every row empty, every page free."""
        self.table.fill_(-1)
        self.lens.fill_(-1)
        self.refs.zero_()
        self.status.zero_()

    def start(self, rows: torch.Tensor) -> None:
        """Rows of a bool mask [rows] that hold no sequence begin one of no tokens."""
        self.lens.copy_(torch.where(rows & (self.lens < 0), 0, self.lens))

    def update(self, parent: Optional[torch.Tensor] = None, n_new: int = 0, advance: int = 0) -> None:
        """ops.paged_update on this cache: fork by parent, lens += advance, make the
        next n_new tokens writable."""
        ops.paged_update(self.k_pages, self.v_pages, self.table, self.lens, self.refs, self.status, parent, n_new,
                         advance)

    def free(self, rows: torch.Tensor) -> None:
        """Rows of a bool mask [rows] let go of their pages and hold no sequence."""
        at = torch.arange(self.rows, dtype=torch.int32, device=self.lens.device)
        self.update(parent=torch.where(rows, -1, at).to(torch.int32))

    def load(self, k_rows: torch.Tensor, v_rows: torch.Tensor, first: torch.Tensor, last: torch.Tensor) -> None:
        """ops.paged_write: positions first[r] .. last[r] - 1 of dense rows [layers,
        rows, kv_heads, positions, head_dim] into pages that update made writable."""
        ops.paged_write(self.k_pages, self.v_pages, self.table, k_rows, v_rows, first, last)

    def attend(self, layer: int, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               want_kctx: bool = True) -> List[Optional[torch.Tensor]]:
        """ops.paged_decode_step of one layer."""
        return ops.paged_decode_step(qkv, self.k_pages[layer], self.v_pages[layer], self.table, self.lens, cos, sin,
                                     want_kctx)

    def compact(self) -> int:
        """Move the pages in use to the lowest ids; returns their number (a host sync)."""
        ops.paged_compact(self.k_pages, self.v_pages, self.table, self.refs, self._used)
        return int(self._used)

    def check(self) -> None:
        """Raise if an update since the last reset found no page (a host sync)."""
        n = int(self.status)
        if n:
            raise RuntimeError(f"paged cache: {n} pages could not be had ({self.n_pages} pages of {self.page_size} tokens); "
                               "rows without their page gave NaN")

    def workspace(self, q_heads: int) -> torch.Tensor:
        """Scratch for loom_paged_decode_step on this cache, for callers of the C entry
        point that keep their own buffers."""
        _, _, kvh, ps, hd = self.k_pages.shape
        with torch.cuda.device(self.k_pages.device):
            n = _lib.load().loom_paged_decode_workspace_bytes(self.rows, self.table.shape[1] * ps, q_heads, kvh, hd)
        return torch.empty((n + 3) // 4, dtype=torch.float32, device=self.k_pages.device)
