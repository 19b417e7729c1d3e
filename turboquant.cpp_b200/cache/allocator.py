"""Host-side bookkeeping of the cache: pages of key/value storage and slots of fixed-size state.

Nothing here touches a device, so the rules can be tested on a CPU: a page or a slot is held by
at most one sequence, is given back exactly once, and none is lost.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence


class CacheFull(RuntimeError):
    """The cache cannot hold what a step asks for."""


class CacheMisuse(RuntimeError):
    """A page or slot was given back twice, or by someone who does not hold it."""


class IndexPool:
    """A pool of indices 0..n-1.  Freed indices are used again, most recently freed first."""

    def __init__(self, n: int, what: str):
        self.n, self.what = int(n), what
        self._free: List[int] = list(range(self.n - 1, -1, -1))
        self._held = [False] * self.n

    @property
    def n_free(self) -> int:
        return len(self._free)

    @property
    def n_held(self) -> int:
        return self.n - len(self._free)

    def take(self) -> int:
        if not self._free:
            raise CacheFull(f"no free {self.what} (all {self.n} are held)")
        i = self._free.pop()
        self._held[i] = True
        return i

    def take_many(self, count: int) -> List[int]:
        if count > len(self._free):
            raise CacheFull(f"{count} {self.what}s wanted, {len(self._free)} of {self.n} are free")
        return [self.take() for _ in range(count)]

    def give_back(self, i: int) -> None:
        if not 0 <= i < self.n:
            raise CacheMisuse(f"{self.what} {i} does not exist (0..{self.n - 1})")
        if not self._held[i]:
            raise CacheMisuse(f"{self.what} {i} is given back but not held")
        self._held[i] = False
        self._free.append(i)

    def is_held(self, i: int) -> bool:
        return self._held[i]


class Sequence_:
    """One live sequence: its slot, its length and, for each group of layers, its pages
    (index = position // page_size; None where a windowed group has given a page back)."""

    def __init__(self, seq_id: int, slot: int, n_groups: int):
        self.id = seq_id
        self.slot = slot
        self.length = 0                  # tokens: the next one's position
        self.evicted = 0                 # of them, those whose rows were given up
        self.pages: List[List[Optional[int]]] = [[] for _ in range(n_groups)]
        self.open = True

    @property
    def held(self) -> int:
        """Rows the sequence holds in the cache: the place of its next token."""
        return self.length - self.evicted


class CacheBook:
    """Pages and slots of all groups.  ``windows[g]`` is the window of group g (0: keeps all);
    ``keep_first[g]`` positions at a sequence's start stay in a windowed group for good."""

    def __init__(self, n_pages: Sequence[int], windows: Sequence[int], page_size: int, max_slots: int,
                 keep_first: Optional[Sequence[int]] = None):
        assert len(n_pages) == len(windows)
        self.page_size = int(page_size)
        self.windows = [int(w) for w in windows]
        self.keep_first = [int(k) for k in keep_first] if keep_first is not None else [0] * len(self.windows)
        assert len(self.keep_first) == len(self.windows)
        self.pools = [IndexPool(n, f"page of group {g}") for g, n in enumerate(n_pages)]
        self.slots = IndexPool(max_slots, "sequence slot")
        self.spare: List[List[int]] = [[] for _ in self.pools]      # pages no sequence holds, for moves (keep_spare)
        self.n_spare = 0                                            # how many of each group there are between moves
        self._next_id = 0
        self.live: Dict[int, Sequence_] = {}

    def open(self) -> Sequence_:
        s = Sequence_(self._next_id, self.slots.take(), len(self.pools))
        self._next_id += 1
        self.live[s.id] = s
        return s

    def pages_needed(self, seq: Sequence_, n_new: int) -> List[int]:
        total = -(-(seq.held + n_new) // self.page_size)
        return [max(0, total - len(p)) for p in seq.pages]

    def reserve(self, seq: Sequence_, n_new: int) -> None:
        """Pages so that positions length .. length+n_new-1 can be written.  All or nothing."""
        self._check_open(seq)
        need = self.pages_needed(seq, n_new)
        for g, c in enumerate(need):
            if c > self.pools[g].n_free:
                raise CacheFull(f"sequence {seq.id} needs {c} more pages of {self.page_size} tokens in group {g} "
                                f"for {seq.held}+{n_new} tokens, {self.pools[g].n_free} of {self.pools[g].n} are free")
        for g, c in enumerate(need):
            seq.pages[g].extend(self.pools[g].take_many(c))

    def reserve_all(self, seqs: Sequence[Sequence_], n_new: Sequence[int]) -> None:
        """Reserve for a whole step, or for none of it."""
        for g in range(len(self.pools)):
            want = sum(self.pages_needed(s, n)[g] for s, n in zip(seqs, n_new))
            if want > self.pools[g].n_free:
                raise CacheFull(f"the step needs {want} more pages of {self.page_size} tokens in group {g}, "
                                f"{self.pools[g].n_free} of {self.pools[g].n} are free")
        for s, n in zip(seqs, n_new):
            self.reserve(s, n)

    def commit(self, seq: Sequence_, n_new: int) -> None:
        """The step wrote n_new tokens.  A windowed group gives back the pages no later query can see:
        a query at position p >= length reads positions >= p + 1 - window, and the group's first keep_first
        positions (their pages are never given back)."""
        self._check_open(seq)
        seq.length += n_new
        for g, w in enumerate(self.windows):
            if w <= 0:
                continue
            first_visible = max(0, seq.length + 1 - w)
            kept = -(-self.keep_first[g] // self.page_size)
            for i in range(kept, min(first_visible // self.page_size, len(seq.pages[g]))):
                if seq.pages[g][i] is not None:
                    self.pools[g].give_back(seq.pages[g][i])
                    seq.pages[g][i] = None

    # ---- eviction: a sequence's rows move to other pages, and there are fewer of them --------------
    def keep_spare(self, rows: int) -> None:
        """Sets pages for `rows` rows aside in every group, so that one sequence can always be moved."""
        self.n_spare = -(-int(rows) // self.page_size)
        self.spare = [pool.take_many(self.n_spare) for pool in self.pools]

    def take_for_moves(self, n: int, rows: int) -> List[List[List[int]]]:
        """New pages for `rows` rows each of up to n sequences (as many as the free pages allow, at least one): per sequence, per group.
        Follow with `moved` for each of them, or with `not_moved`."""
        per = -(-int(rows) // self.page_size)
        if any(len(s) < per for s in self.spare):
            raise CacheMisuse(f"no pages for {rows} rows are set aside")
        first = [s[:per] for s in self.spare]
        self.spare = [s[per:] for s in self.spare]
        out = [first]
        while len(out) < n and all(pool.n_free >= per for pool in self.pools):
            out.append([pool.take_many(per) for pool in self.pools])
        return out

    def moved(self, seq: Sequence_, pages: List[List[int]], rows: int) -> None:
        """The sequence now holds `rows` rows, on these pages; its old ones are set aside again or free."""
        self._check_open(seq)
        for g, new in enumerate(pages):
            self._give_back(g, seq.pages[g])
            seq.pages[g] = list(new)
        seq.evicted = seq.length - rows

    def not_moved(self, pages: List[List[int]]) -> None:
        """Pages of `take_for_moves` that no sequence moved to are set aside again or free."""
        for g, back in enumerate(pages):
            self._give_back(g, back)

    def _give_back(self, g: int, pages: List[int]) -> None:
        for p in pages:
            if len(self.spare[g]) < self.n_spare:
                self.spare[g].append(p)
            else:
                self.pools[g].give_back(p)
        # (a sequence of fewer pages than it moved to)
        self.spare[g] += self.pools[g].take_many(min(self.n_spare - len(self.spare[g]), self.pools[g].n_free))

    def close(self, seq: Sequence_) -> None:
        self._check_open(seq)
        for g, pages in enumerate(seq.pages):
            for p in pages:
                if p is not None:
                    self.pools[g].give_back(p)
            pages.clear()
        self.slots.give_back(seq.slot)
        seq.open = False
        del self.live[seq.id]

    def _check_open(self, seq: Sequence_) -> None:
        if not seq.open or self.live.get(seq.id) is not seq:
            raise CacheMisuse(f"sequence {seq.id} is not live in this cache (closed twice?)")

    def check_invariants(self) -> None:
        """Every page and slot is either free or held by exactly one live sequence."""
        for g, pool in enumerate(self.pools):
            held = [p for s in self.live.values() for p in s.pages[g] if p is not None] + self.spare[g]
            if len(held) != len(set(held)):
                raise AssertionError(f"group {g}: a page is held twice")
            if len(held) != pool.n_held:
                raise AssertionError(f"group {g}: {pool.n_held} pages are out but sequences hold {len(held)}")
        slots = [s.slot for s in self.live.values()]
        if len(slots) != len(set(slots)) or len(slots) != self.slots.n_held:
            raise AssertionError("slots held do not match live sequences")
