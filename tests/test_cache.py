"""The cache's bookkeeping (CPU): no page or slot lost, held twice or freed twice."""
import random

import pytest
import torch

from turboquant_cpp_b200.cache import CacheBook, CacheFull, CacheMisuse, IndexPool, PagedCache
from turboquant_cpp_b200.parts import KVNeed, StateNeed


def test_pool_gives_each_index_once_and_takes_it_back_once():
    p = IndexPool(4, "page")
    got = [p.take() for _ in range(4)]
    assert sorted(got) == [0, 1, 2, 3]
    with pytest.raises(CacheFull):
        p.take()
    p.give_back(got[1])
    with pytest.raises(CacheMisuse):
        p.give_back(got[1])                      # freed twice
    with pytest.raises(CacheMisuse):
        p.give_back(17)
    assert p.take() == got[1]                    # used again


def test_sequences_reserve_commit_close():
    book = CacheBook([8, 8], [0, 0], page_size=64, max_slots=3)
    a, b = book.open(), book.open()
    assert a.slot != b.slot
    book.reserve_all([a, b], [70, 1])
    assert [len(x) for x in a.pages] == [2, 2] and [len(x) for x in b.pages] == [1, 1]
    book.commit(a, 70)
    book.commit(b, 1)
    book.reserve(a, 58)                          # 70 + 58 = 128: still two pages
    assert len(a.pages[0]) == 2
    book.commit(a, 58)
    book.reserve(a, 1)
    assert len(a.pages[0]) == 3
    book.check_invariants()
    book.close(a)
    with pytest.raises(CacheMisuse):
        book.close(a)                            # closed twice
    with pytest.raises(CacheMisuse):
        book.reserve(a, 1)
    book.close(b)
    book.check_invariants()
    assert all(p.n_free == 8 for p in book.pools) and book.slots.n_free == 3


def test_reserve_all_is_all_or_nothing():
    book = CacheBook([3], [0], page_size=64, max_slots=4)
    a, b = book.open(), book.open()
    with pytest.raises(CacheFull):
        book.reserve_all([a, b], [128, 128])     # 4 pages wanted, 3 there
    assert book.pools[0].n_free == 3 and not a.pages[0] and not b.pages[0]
    book.reserve_all([a, b], [128, 64])
    assert book.pools[0].n_free == 0
    c = book.open()
    with pytest.raises(CacheFull):
        book.reserve(c, 1)
    with pytest.raises(CacheFull):
        [book.open() for _ in range(2)]          # slots run out too
    book.check_invariants()


def test_windowed_group_gives_old_pages_back():
    book = CacheBook([10, 10], [0, 32], page_size=64, max_slots=2)
    s = book.open()
    book.reserve(s, 200)
    book.commit(s, 200)                          # later queries see positions >= 201 - 32 = 169: pages 0, 1 go
    assert [p is None for p in s.pages[1]] == [True, True, False, False]
    assert all(p is not None for p in s.pages[0])
    assert book.pools[1].n_free == 8 and book.pools[0].n_free == 6
    book.reserve(s, 100)
    book.commit(s, 100)                          # 300 tokens: positions >= 269: pages 0..3 gone
    assert [p is None for p in s.pages[1]] == [True] * 4 + [False]
    book.check_invariants()
    book.close(s)
    assert book.pools[1].n_free == 10


def test_random_walk_keeps_the_books():
    rng = random.Random(0)
    book = CacheBook([40, 40], [0, 100], page_size=64, max_slots=6)
    live = []
    for _ in range(2000):
        r = rng.random()
        try:
            if r < 0.2 and len(live) < 6:
                live.append(book.open())
            elif r < 0.8 and live:
                s = rng.choice(live)
                n = rng.choice([1, 1, 1, 5, 64, 130])
                book.reserve(s, n)
                book.commit(s, n)
            elif live:
                book.close(live.pop(rng.randrange(len(live))))
        except CacheFull:
            if live:
                book.close(live.pop(0))
        book.check_invariants()
    for s in live:
        book.close(s)
    assert all(p.n_free == p.n for p in book.pools) and book.slots.n_free == 6


def test_paged_cache_groups_state_and_tables():
    full, win = KVNeed(2, 16, 0), KVNeed(2, 16, 32)
    needs = [full, win, None, win, full]          # entry 2 keeps no keys; entry 4 reads entry 0's cache
    state = [None, None, StateNeed((3, 4)), None, None]
    cache = PagedCache(needs, state, [None, None, None, None, 0], max_tokens=640, dtype=torch.float32, device="cpu",
                       max_slots=4)
    assert cache.groups == [full, win] and cache.entry_group == [0, 1, None, 1, 0]
    assert cache.kv[4] is cache.kv[0] and cache.kv[2] is None
    assert cache.kv[0].shape == (10, 2, 2, 64, 16) and cache.kv[1] is not cache.kv[3]
    assert cache.state[2].shape == (4, 3, 4)
    a = cache.open()
    cache.state[2][a.slot] += 1.0
    cache.reserve([a], [130])
    cache.commit([a], [130])
    t = cache.page_tables([a])
    assert t[0].shape == (1, 3) and (t[0] >= 0).all()
    assert t[1].tolist()[0][0] == -1 and t[1].tolist()[0][2] >= 0      # window 32: page 0 was given back
    lc = cache.layer_caches([torch.from_numpy(x) for x in t])
    assert lc[4].writes is False and lc[0].writes is True and lc[2].kv is None and lc[2].state is cache.state[2]
    slot = a.slot
    cache.close(a)
    b = cache.open()
    assert b.slot == slot and float(cache.state[2][slot].abs().sum()) == 0.0     # the slot is used again, zeroed
    assert cache.bytes_per_token() == 3 * 2 * 2 * 16 * 4      # three entries keep keys and values


# ---- sequences that give rows up --------------------------------------------------------------------------------------
def test_moved_sequences_hold_fewer_rows_on_other_pages():
    book = CacheBook([12, 12], [0, 0], page_size=64, max_slots=4)
    book.keep_spare(130)                          # three pages a group set aside
    assert [p.n_free for p in book.pools] == [9, 9]
    book.check_invariants()
    a, b = book.open(), book.open()
    book.reserve_all([a, b], [250, 200])
    book.commit(a, 250)
    book.commit(b, 200)
    assert (a.held, b.held) == (250, 200) and [p.n_free for p in book.pools] == [1, 1]
    old = [list(p) for p in a.pages]
    moves = book.take_for_moves(2, 130)           # one free page: only what is set aside
    assert len(moves) == 1 and all(len(m) == 3 and not set(m) & set(o) for m, o in zip(moves[0], old))
    book.moved(a, moves[0], 130)
    assert (a.held, a.length) == (130, 250) and [len(s) for s in book.spare] == [3, 3] and [p.n_free for p in book.pools] == [2, 2]
    book.check_invariants()
    book.reserve(a, 62)                           # places 130 .. 191: the three pages it has
    assert [len(p) for p in a.pages] == [3, 3]
    book.commit(a, 62)
    book.reserve(a, 1)
    assert a.held == 192 and a.length == 312 and [len(p) for p in a.pages] == [4, 4]
    book.check_invariants()
    book.close(a)
    moves = book.take_for_moves(5, 130)           # free pages serve further sequences of the same step
    assert len(moves) == 2                        # 12 - 3 set aside - 4 of b's: 5 free, room for one more of three
    book.moved(b, moves[0], 130)
    for m in moves[1:]:
        for g, pages in enumerate(m):
            for p in pages:
                book.pools[g].give_back(p)
    book.check_invariants()
    book.close(b)
    assert [p.n_free for p in book.pools] == [9, 9]
    with pytest.raises(CacheMisuse):
        book.take_for_moves(1, 500)               # more than was set aside


def test_batches_count_bounded_requests_by_what_they_come_to_hold():
    from turboquant_cpp_b200.engine.generate import plan_batches
    plan = lambda bounded: plan_batches([100, 100, 900, 10], 4000, 8, 2048, 8, 64, 8192, bounded)
    assert plan(0) == [[0], [1], [2], [3]]
    assert plan(256) == [[0, 1, 2, 3]]            # 256, 256, its prompt of 900, 256: 27 of 32 pages
    assert plan_batches([100, 100], 20, 8, 256, 8, 64, 8192, 4096) == [[0, 1]]


def test_options_that_an_engine_refuses(monkeypatch):
    """Checked before anything is built: no GPU."""
    import turboquant_cpp_b200 as tq
    from conftest import TINY_A, TINY_B
    import copy
    import lumevik_util
    make = lambda cfg: tq.build_model(cfg, "bfloat16")
    check = lambda model, dtype, budget=0, recent=None: _engine_options(model, dtype, budget, recent)
    odd = copy.deepcopy(TINY_A)
    assert check(make(odd), "e4m3") is True and check(make(odd), "") is False and check(make(odd), "e4m3", 64) is True
    assert check(make(TINY_B), "e4m3") is True
    for model, dtype, budget, recent in ((make(odd), "int4", 0, None), (make(odd), "", 64, None), (make(odd), "e4m3", 64, 65), (make(odd), "e4m3", -1, None),
                                         (make(TINY_B), "e4m3", 64, None), (make(next(iter(lumevik_util.CONFIGS.values()))), "e4m3", 0, None)):
        with pytest.raises(ValueError):
            check(model, dtype, budget, recent)


def _engine_options(model, dtype, budget, recent):
    from turboquant_cpp_b200.engine.step import Engine
    e = Engine.__new__(Engine)
    e.cache_budget, e.cache_recent = budget, budget // 4 if recent is None else recent
    return e._cache_in_8_bits(model, dtype)


def test_the_pages_set_aside_stay_as_many():
    """Moves to fewer pages than are set aside, and of sequences that hold fewer than they move to: the next move still finds its pages."""
    book = CacheBook([20], [0], page_size=64, max_slots=4)
    book.keep_spare(256)                          # four pages
    for length, rows in ((500, 64), (100, 100), (70, 256), (300, 130), (600, 256)):
        seq = book.open()
        book.reserve(seq, length)
        book.commit(seq, length)
        (pages,) = book.take_for_moves(1, rows)
        book.moved(seq, pages, min(rows, length))
        assert len(book.spare[0]) == 4 and seq.held == min(rows, length), (length, rows)
        book.check_invariants()
        book.close(seq)
    assert book.pools[0].n_free == 16


def test_an_eviction_that_fails_gives_its_pages_back(monkeypatch):
    """Its sequences stay as they were: the old pages are only read."""
    import numpy as np
    from turboquant_cpp_b200.cache import paged
    cache = PagedCache([KVNeed(1, 16)], [None], [None], 640, torch.bfloat16, "cpu", eight_bits=True, weights=True)
    cache.book.keep_spare(64)
    seq = cache.open()
    cache.reserve([seq], [200])
    cache.commit([seq], [200])
    pages, free = [list(p) for p in seq.pages], cache.book.pools[0].n_free

    def fails(*a):
        raise RuntimeError("no")
    monkeypatch.setattr(paged, "evict8", fails)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    for seqs in ([seq], [seq, seq]):
        with pytest.raises(RuntimeError, match="no"):
            cache.evict(seqs, 64, 4)
        assert seq.pages == pages and seq.held == 200 and len(cache.book.spare[0]) == 1 and cache.book.pools[0].n_free == free
        cache.book.check_invariants()
    kept = []
    monkeypatch.setattr(paged, "evict8", lambda codes, scales, weights, lengths, *a: kept.append(lengths.tolist()))
    short = cache.open()
    cache.reserve([short], [64])
    cache.commit([short], [64])
    mine = [list(p) for p in short.pages]
    cache.evict([short, seq], 64, 4)
    assert kept == [[200]] and (seq.held, short.held) == (64, 64) and short.pages == mine        # within the budget: nothing to give up
    cache.book.check_invariants()


def test_bytes_of_a_token_where_groups_have_pages_of_their_own():
    """An 8-bit row's scales and sums count by the pages of their own group."""
    near, far = KVNeed(2, 32, window=64), KVNeed(4, 16)
    cache = PagedCache([near, far], [None, None], [None, None], 640, torch.bfloat16, "cpu", pages_per_group={near: 2, far: 40}, eight_bits=True, weights=True)
    assert cache.bytes_per_token() == 2 * 2 * 32 + 2 * 4 * 16 + -(-2 * (2 + 4) // 16) + 4 * (2 + 4)
