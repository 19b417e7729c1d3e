"""The cache on the device: pages of keys and values for every layer that keeps some, in groups
of layers with equal needs, and an area of fixed-size state per sequence slot.

The reference keeps one sequence's keys and values as [layer][position][kv heads * head size]
arrays written at the token's position (src/engine/tq_transformer.c:210-227, 1371, 1452-1455) and
its recurrent layers' fixed-size state in the same object, zeroed at creation
(include/turboquant/tq_engine.h:329-330; src/engine/tq_transformer.c:291-313).  Here:

* a *group* is the set of schedule entries whose mixers have the same KVNeed (heads, head size,
  window).  Each group has its own pool of pages and each sequence its own page list per group,
  so layers that keep every key and layers that keep a window of them are stored apart; a
  windowed group gives pages back as they fall out of every later query's sight.
* an entry's storage is one tensor [pages, planes, kv heads, page_size, head size]: two planes (K, V), or one
  for a mixer whose cached row serves as key and value.
* in 8 bits (`eight_bits`) an entry's storage is codes and their blocks' bytes (kernels/cache8.py) and, where sequences are evicted by
  it (`weights`), the attention weight every row has received.  A sequence that was evicted holds fewer rows than tokens: a row's
  place in its pages is then no longer its position.
* a sequence holds a *slot*: its row in every state tensor [max_slots, *shape].  The row is
  zeroed when the slot is taken.  Slots and pages are given back when the sequence is closed and
  are used again by later sequences.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels.cache8 import BLOCK, evict8, storage as storage8
from ..parts.base import KVNeed, LayerCache, StateNeed
from .allocator import CacheBook, CacheFull, Sequence_

PAGE_SIZE = 64


class PagedCache:
    def __init__(self, kv_needs: Sequence[Optional[KVNeed]], state_needs: Sequence[Optional[StateNeed]],
                 cache_of: Sequence[Optional[int]], max_tokens: int, dtype: torch.dtype, device,
                 max_slots: Optional[int] = None, page_size: int = PAGE_SIZE,
                 pages_per_group: Optional[Dict[KVNeed, int]] = None,
                 embed_state_need: Optional[StateNeed] = None, eight_bits: bool = False, weights: bool = False):
        """kv_needs/state_needs/cache_of: one item per entry of the model's layer schedule.
        max_tokens: the most tokens live sequences hold together, each sequence's count rounded up
        to a multiple of page_size."""
        self.page_size = int(page_size)
        self.device = torch.device(device)
        self.dtype = dtype
        self.eight_bits = bool(eight_bits)
        n_pages = max(1, -(-int(max_tokens) // self.page_size))
        self.max_slots = int(max_slots) if max_slots is not None else min(n_pages, 1024)
        self.groups: List[KVNeed] = []
        self.entry_group: List[Optional[int]] = []
        for i, need in enumerate(kv_needs):
            src = cache_of[i]
            if src is not None:
                self.entry_group.append(None)      # filled below from its source
                continue
            if need is None:
                self.entry_group.append(None)
                continue
            if need not in self.groups:
                self.groups.append(need)
            self.entry_group.append(self.groups.index(need))
        for i, src in enumerate(cache_of):
            if src is not None:
                self.entry_group[i] = self.entry_group[src]
        counts = [(pages_per_group or {}).get(g, n_pages) for g in self.groups]
        self.book = CacheBook(counts, [g.window for g in self.groups], self.page_size, self.max_slots,
                              keep_first=[g.keep_first for g in self.groups])
        self.kv: List[Optional[torch.Tensor]] = []
        self.scales: List[Optional[torch.Tensor]] = [None] * len(kv_needs)
        self.weights: List[Optional[torch.Tensor]] = [None] * len(kv_needs)
        for i, need in enumerate(kv_needs):
            if need is None or cache_of[i] is not None:
                self.kv.append(None)
                continue
            g = self.entry_group[i]
            if eight_bits:
                if need.planes != 2:
                    raise ValueError("a cache in 8 bits keeps keys and values, not rows that serve as both")
                codes, self.scales[i], self.weights[i] = storage8(counts[g], need.n_kv_heads, self.page_size, need.head_dim, self.device, weights)
                self.kv.append(codes)
                continue
            self.kv.append(torch.zeros((counts[g], need.planes, need.n_kv_heads, self.page_size, need.head_dim),
                                       dtype=dtype, device=self.device))
        for i, src in enumerate(cache_of):
            if src is not None:
                self.kv[i], self.scales[i], self.weights[i] = self.kv[src], self.scales[src], self.weights[src]
        self.cache_of = list(cache_of)
        self.state: List[Optional[torch.Tensor]] = [
            None if n is None else torch.zeros((self.max_slots,) + tuple(n.shape), dtype=n.dtype, device=self.device)
            for n in state_needs]
        # state the embedding keeps per sequence (a design whose embedding looks at the token before)
        self.embed_state: Optional[torch.Tensor] = None if embed_state_need is None else torch.zeros(
            (self.max_slots,) + tuple(embed_state_need.shape), dtype=embed_state_need.dtype, device=self.device)

    # ---- sequences ------------------------------------------------------------------------------
    def open(self) -> Sequence_:
        seq = self.book.open()
        for s in self.state + [self.embed_state]:
            if s is not None:
                s[seq.slot].zero_()
        return seq

    def close(self, seq: Sequence_) -> None:
        self.book.close(seq)

    def reserve(self, seqs: Sequence[Sequence_], n_new: Sequence[int]) -> None:
        self.book.reserve_all(seqs, n_new)

    def commit(self, seqs: Sequence[Sequence_], n_new: Sequence[int]) -> None:
        for s, n in zip(seqs, n_new):
            self.book.commit(s, n)

    # ---- what a step sees -----------------------------------------------------------------------
    def page_tables(self, seqs: Sequence[Sequence_]) -> List[np.ndarray]:
        """Per group an int32 array [n_seqs, width]: the pages of each sequence (-1: none)."""
        out = []
        for g in range(len(self.groups)):
            width = max(1, max((len(s.pages[g]) for s in seqs), default=1))
            t = np.full((len(seqs), width), -1, dtype=np.int32)
            for i, s in enumerate(seqs):
                pages = s.pages[g]
                if pages:
                    t[i, :len(pages)] = [(-1 if p is None else p) for p in pages]
            out.append(t)
        return out

    def layer_caches(self, device_tables: Sequence[torch.Tensor]) -> List[LayerCache]:
        out = []
        for i in range(len(self.kv)):
            g = self.entry_group[i]
            out.append(LayerCache(kv=self.kv[i], page_table=None if g is None else device_tables[g],
                                  page_size=self.page_size, writes=self.cache_of[i] is None,
                                  state=self.state[i], scales=self.scales[i], weights=self.weights[i]))
        return out

    def bytes_per_token(self) -> int:
        """Key/value bytes one token adds across all layers that keep a cache."""
        own = [i for i, t in enumerate(self.kv) if t is not None and self.cache_of[i] is None]
        rows = sum(self.kv[i].shape[1] * self.kv[i].shape[2] * self.kv[i].shape[4] * self.kv[i].element_size() for i in own)
        if not self.eight_bits:
            return rows
        scales = sum(2 * self.kv[i].shape[2] for i in own)                      # a byte each for BLOCK rows
        return rows + -(-scales // BLOCK) + sum(4 * self.kv[i].shape[2] for i in own if self.weights[i] is not None)

    # ---- eviction -------------------------------------------------------------------------------
    def evict(self, seqs: Sequence[Sequence_], budget: int, recent: int) -> None:
        """The sequences that hold more than `budget` rows keep that many in every key/value head of every layer (kernels.cache8.evict8), on pages of
        their own.  An error leaves those that were not done as they were."""
        todo = [s for s in seqs if s.held > budget]
        while todo:
            moves = self.book.take_for_moves(len(todo), budget)
            now, todo = todo[:len(moves)], todo[len(moves):]
            try:
                self._evict_to(now, moves, budget, recent)
            except BaseException:
                for m in moves:
                    self.book.not_moved(m)
                raise
            for s, m in zip(now, moves):
                self.book.moved(s, m, budget)

    def _evict_to(self, now: Sequence[Sequence_], moves, budget: int, recent: int) -> None:
        tables = self.page_tables(now)
        fields = [np.array([s.held for s in now], dtype=np.int32)] + tables + [np.array([m[g] for m in moves], dtype=np.int32) for g in range(len(self.groups))]
        sizes = [f.size for f in fields]
        parts = torch.split(torch.from_numpy(np.concatenate([f.reshape(-1) for f in fields])).pin_memory().to(self.device, non_blocking=True), sizes)
        for i, codes in enumerate(self.kv):
            if codes is None or self.cache_of[i] is not None:
                continue
            g = self.entry_group[i]
            evict8(codes, self.scales[i], self.weights[i], parts[0], parts[1 + g].view(tables[g].shape),
                   parts[1 + len(self.groups) + g].view(len(now), -1), self.page_size, budget, recent)
