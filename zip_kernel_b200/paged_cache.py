"""Paged key/value cache of a decoder stack: the pages of all layers, one block table and the lengths they share.

A serving loop calls :meth:`PagedKVCache.advance` once per step, passes :meth:`PagedKVCache.layer` and the shared
``lengths`` / ``offsets`` to the operators of :mod:`zip_kernel_b200.paged_ops` in every layer, and now and then shortens
all histories with :meth:`PagedKVCache.evict`.  Everything that a step changes is on the device and changed in place, so a
decode step can be captured in a CUDA graph and replayed.  No counterpart in the reference.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops


class PagedKVCache:
    """``n_seqs`` sequences of up to ``max_slots`` slots in every one of ``n_layers`` layers.

    ``lengths (n_seqs)`` int32: slots in use; ``offsets (n_seqs)`` int32: slots evicted so far, so that position = slot + offset;
    ``sums (n_layers, n_seqs, n_kv_heads, slots)`` float32 with ``track_weights=True``: attention weight received, which
    :meth:`add_weights` adds up and :meth:`evict` goes by."""

    def __init__(self, n_layers: int, n_seqs: int, max_slots: int, n_kv_heads: int, head_dim: int, *, page_size: int = 64,
                 dtype=torch.float16, device="cuda", track_weights: bool = False):
        if n_layers < 1 or n_seqs < 1 or max_slots < 1:
            raise ValueError(f"layers ({n_layers}), sequences ({n_seqs}) and slots ({max_slots}) must be positive")
        if page_size < 16 or page_size % 16:
            raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
        cols = (max_slots + page_size - 1) // page_size
        n_pages = n_seqs * cols
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.device = self.k_pages.device
        self.n_layers, self.n_seqs, self.max_slots = int(n_layers), int(n_seqs), cols * page_size
        self.block_table = torch.arange(n_pages, dtype=torch.int32, device=self.device).reshape(n_seqs, cols)
        self.layers = [ops.PagedKV(self.k_pages[i], self.v_pages[i], self.block_table) for i in range(n_layers)]
        # all layers as one cache of n_layers * n_seqs sequences, for the eviction
        table = self.block_table + n_pages * torch.arange(n_layers, dtype=torch.int32, device=self.device)[:, None, None]
        self._all = ops.PagedKV(self.k_pages.flatten(0, 1), self.v_pages.flatten(0, 1), table.reshape(n_layers * n_seqs, cols).contiguous())
        self.lengths = torch.zeros(n_seqs, dtype=torch.int32, device=self.device)
        self.offsets = torch.zeros(n_seqs, dtype=torch.int32, device=self.device)
        self.sums: Optional[torch.Tensor] = None
        if track_weights:
            self.sums = torch.zeros((n_layers, n_seqs, n_kv_heads, self.max_slots), dtype=torch.float32, device=self.device)
        self._ones = torch.arange(n_seqs + 1, dtype=torch.int32, device=self.device)

    def layer(self, i: int) -> ops.PagedKV:
        return self.layers[i]

    def cu_seqlens(self, q_len: int) -> torch.Tensor:
        """Offsets of a step in which every sequence has ``q_len`` new tokens.  Made on the current stream at every call, but for
        the one of single tokens: a tensor kept from a capture would be empty until the graph's first replay."""
        return self._ones if q_len == 1 else self._ones * q_len

    def advance(self, q_len: int) -> torch.Tensor:
        """Makes room for ``q_len`` new tokens of every sequence (once per step, before its first layer) and returns the
        step's ``cu_seqlens``.  The caller keeps the lengths within ``max_slots``."""
        self.lengths.add_(q_len)
        return self.cu_seqlens(q_len)

    def add_weights(self, i: int, q: torch.Tensor, lse: torch.Tensor, cu_seqlens: torch.Tensor, max_q_len: int) -> None:
        """Adds the attention weight of these queries to layer ``i``'s sums."""
        if self.sums is None:
            raise RuntimeError("the cache was made without track_weights")
        ops.cache_weight_sums_cuda(q, self.layers[i], cu_seqlens, self.lengths, lse, self.sums[i], max_q_len=max_q_len)

    def evict(self, budget: int, *, n_sink: int = 0, n_recent: int = 0) -> torch.Tensor:
        """Shortens every sequence to at most ``budget`` slots in every layer and head (see
        :func:`~zip_kernel_b200.paged_ops.cache_evict_cuda`) and returns the old slot of each kept one,
        ``(n_layers, n_seqs, n_kv_heads, budget)`` int32."""
        if self.sums is None:
            raise RuntimeError("the cache was made without track_weights")
        kept, new, sums = ops.cache_evict_cuda(self._all, self.lengths.repeat(self.n_layers), self.sums.flatten(0, 1), budget,
                                               n_sink=n_sink, n_recent=n_recent)
        new = new[:self.n_seqs]
        self.offsets.add_(self.lengths - new)
        self.lengths.copy_(new)
        self.sums.copy_(sums.view_as(self.sums))
        return kept.view(self.n_layers, self.n_seqs, *kept.shape[1:])


__all__ = ["PagedKVCache"]
