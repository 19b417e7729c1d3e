"""Calls of the 8-bit cache that its documentation allows at the edges of its ranges: weights far below the largest, tensors off their 16-byte
boundaries, plans made for longer sequences than there are, steps dropped, against plain implementations in 64 bits."""
import math

import pytest
import torch

from plain import cache8_plain as plain
from test_cache8_gpu import DEV, U, _attend, _cache, _cu, _i, _limit, _on, _pages

pytestmark = pytest.mark.gpu


def _sinks(rows, D, value_of):
    """A cache of one sequence and one key/value head: of every 16 rows the first has key e0 and value 0, the others key 0 and values of value_of(shape).
    With the query e0 the first score `scale`, the others 0."""
    table, pages = _pages([rows], 64)
    codes, scales = torch.zeros(pages, 2, 1, 64, D, dtype=torch.uint8), torch.full((pages, 2, 1, 4), 127, dtype=torch.uint8)
    x = value_of((pages, 64, D))
    x[:, ::16] = 0.0
    codes[:, 0, 0, ::16, 0] = torch.ones(1).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[:, 1, 0] = x.to(torch.float8_e4m3fn).view(torch.uint8)
    return table, codes, scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ranges", [1, 3, 12])
@pytest.mark.parametrize("units", [4000.5, 40.5, 5.4, 1.45, 0.45])
def test_many_weights_far_below_the_largest(dtype, D, ranges, units, monkeypatch):
    """Rows whose weight is `units` times 2^-24 of their neighbours' that have no value: the result is theirs alone.  All values are positive, so every
    error is relative to the result: scores and sums as in test_cache8_gpu; a weight of float32 rows is off by 2^-22 of itself and 2^-39 of the largest (two
    parts of 11 bits, multiples of 2^-38), one of bfloat16 rows by half a step of 11 bits."""
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "ranges_for", lambda *a: ranges)
    rows, b = 2000, 24 - math.log2(units)
    table, codes, scales = _sinks(rows, D, lambda shape: 0.5 + torch.rand(shape))
    q = torch.zeros(1, 1, D, dtype=dtype)
    q[0, 0, 0] = 1.0
    scale = float(torch.tensor(b * math.log(2.0)))
    want, mags, sums, _ = plain.attention(q, codes, scales, [1], [rows - 1], table, 64, 0, scale, 1, 1, D)
    got, _ = _attend(q, codes, scales, [1], [rows - 1], table, 64, 0, scale, 1, 1, D)
    weight = 2.0 ** -39 / (units * 2.0 ** -24) + 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    # one product of a score is not 0: its factors are rounded four times, and the exponent is a difference of two scores
    rel = 2.02 * 8 * U * scale * 1.45 + (rows + 16) * 4 * U + weight + torch.finfo(dtype).eps / 2 * (1.01 if dtype == torch.bfloat16 else 8)
    off = (got.double().view(want.shape) - want).abs() / want
    assert float(off.max()) <= rel, (float(off.max()), rel)


@pytest.mark.parametrize("D", [64, 128])
def test_weights_of_single_tokens_have_eleven_bits(D):
    """Weights just above the middle between two numbers of 8 bits: had the kernel of single tokens weights of 8 bits, each of them, and so the result
    ahead of its own rounding, would be off by 2^-8."""
    rows, mantissa = 1000, 1.0 + 2.0 ** -8 * 0.98
    table, codes, scales = _sinks(rows, D, lambda shape: 0.5 + torch.rand(shape))
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16)
    q[0, 0, 0] = 1.0
    scale = float(torch.tensor((12 - math.log2(mantissa)) * math.log(2.0)))
    want, *_ = plain.attention(q, codes, scales, [1], [rows - 1], table, 64, 0, scale, 1, 1, D)
    got, _ = _attend(q, codes, scales, [1], [rows - 1], table, 64, 0, scale, 1, 1, D)
    rel = 2.02 * 8 * U * scale * 1.45 + (rows + 16) * 4 * U + 2.0 ** -11 + 2.0 ** -8 * 1.001
    off = (got.double().view(want.shape) - want).abs() / want
    assert float(off.max()) <= rel, (float(off.max()), rel)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e4, 1e6, 6e7])
@pytest.mark.parametrize("ranges", [1, 5, 12])
def test_scores_far_from_zero(dtype, size, ranges, monkeypatch):
    """All of a row's scores lie `size` above or below zero, exactly: a softmax does not see it."""
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "ranges_for", lambda *a: ranges)
    H, G, D, rows = 2, 1, 64, 1500
    table, pages = _pages([rows], 64)
    codes, scales = _cache(pages, G, 64, D, spread=1.0)
    codes[:, 0] = 0
    codes[:, 0, :, :, 0] = torch.ones(1).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[:, 0] = 127
    want = None
    for sign in (0.0, 1.0, -1.0):
        q = torch.zeros(1, H, D, dtype=dtype)
        q[:, :, 0] = sign
        got, _ = _attend(q, codes, scales, [1], [rows - 1], table, 64, 0, size, H, G, D)
        want = got if want is None else want
        assert torch.equal(got, want), sign


# ---- steps launched ahead ----------------------------------------------------------------------------------------------------
def _begun(model, prompts):
    import turboquant_cpp_b200 as tq
    engine = tq.Engine(model, max_tokens=512, cache_dtype="e4m3")
    seqs = [engine.open() for _ in prompts]
    engine.step([tq.StepEntry(s, p) for s, p in zip(seqs, prompts)])
    engine.step([tq.StepEntry(s, [6], [0]) for s in seqs])
    return engine, seqs


def _rows(engine, seq):
    """The first page of a sequence of up to 16 rows: its codes and bytes, every layer."""
    page = seq.pages[0][0]
    return [t for c, b in zip(engine.cache.kv, engine.cache.scales) for t in (c.view(torch.uint8)[page, :, :, :seq.held].cpu(), b[page, :, :, 0].cpu())]


def test_a_step_launched_ahead_counts_for_those_that_go_on(tiny_folders):
    """A row that raises its block's byte has the rows it finds there rounded again, for good: dropping its step does not undo it.  So the step is kept, and
    leaves what a plain step leaves."""
    import turboquant_cpp_b200 as tq
    from turboquant_cpp_b200.engine.step import StepError
    model = tq.load_model(tiny_folders["A"], "float32", DEV)
    prompts = [[3, 17, 200, 42, 9], [7, 8, 9], [100, 2]]
    (engine, (a, b, c)), (other, theirs) = _begun(model, prompts), _begun(model, prompts)
    before = _rows(engine, a)
    assert engine.can_step_ahead and all(torch.equal(x, y) for x, y in zip(before, _rows(other, theirs[0])))
    for token in range(0, 256, 5):
        tokens = [token, 9, (token + 1) % 256]
        logits = engine.step_ahead([a, b, c], torch.tensor(tokens, dtype=torch.int32, device=DEV)).clone()
        with pytest.raises(StepError):
            engine.drop_ahead()
        with pytest.raises(StepError):
            engine.step([tq.StepEntry(a, [1], [0])])
        with pytest.raises(StepError):
            engine.commit_ahead([a, c])                  # b is open
        if a.held == 10:
            engine.close(b)
            engine.commit_ahead([c, a])
        else:
            engine.commit_ahead()
        want = other.step([tq.StepEntry(s, [t], [0]) for s, t in zip(theirs, tokens)])
        assert torch.equal(logits, want) and a.held == theirs[0].held
        assert all(torch.equal(x, y) for x, y in zip(_rows(engine, a), _rows(other, theirs[0])))
        if not b.open:
            break
    assert any(not torch.equal(x, y) for x, y in zip(before, [t[:, :, :6] if t.dim() == 4 else t for t in _rows(engine, a)]))        # bytes did grow
    with pytest.raises(StepError):
        engine.step_ahead([a], torch.tensor([1], dtype=torch.int32, device=DEV)), engine.commit_ahead([c])
    engine.close(a)
    engine.drop_ahead()                                  # nobody is left whom it could have changed
    assert torch.isfinite(engine.step([tq.StepEntry(c, [1], [0])])).all()
    engine.close(c)
    engine.cache.book.check_invariants()
    engine.release()
    other.release()


def test_generation_whose_requests_end_early(tiny_folders, monkeypatch):
    """Steps ahead of their tokens or not: the same tokens."""
    import turboquant_cpp_b200 as tq
    model = tq.load_model(tiny_folders["A"], "float32", DEV)
    prompts = [[5, 9, 2], list(range(60)), [1] * 20, [200, 100], [77]]
    out = []
    for graphs in (True, False):
        monkeypatch.setenv("TQ_NO_GRAPHS", "0" if graphs else "1")
        with tq.Model.from_model(model, temperature=0.0, max_tokens=40, context_length=128, max_batch=5, stop_token_ids=list(range(0, 256, 17)), cache_dtype="e4m3") as m:
            assert m.engine.can_step_ahead == graphs
            out.append(m.generate_batch(prompts))
            m.engine.cache.book.check_invariants()
    assert out[0] == out[1] and len({len(t) for t in out[0]}) > 1 and min(len(t) for t in out[0]) < 40


# ---- tensors off their 16-byte boundaries --------------------------------------------------------------------------------------
def _off(t, where):
    """The same elements one element behind a boundary of 16 bytes."""
    if not where:
        return t
    x = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    x.copy_(t)
    assert x.data_ptr() % 16 and x.is_contiguous()
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs,held", [([1, 1], [70, 5]), ([60, 3], [0, 40])])
@pytest.mark.parametrize("q_off,out_off", [(True, False), (False, True), (True, True)])
def test_queries_and_results_may_begin_anywhere(dtype, runs, held, q_off, out_off, monkeypatch):
    """Whatever the step's size: with the long run the prompt kernel is asked for, which itself wants 16-byte boundaries.  Rows behind the last sequence stay."""
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    H, G, D = 8, 2, 64
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D)
    q = torch.randn(sum(runs) + 2, H, D).to(dtype).to(DEV)
    seen = []
    for moved in (False, True):
        out = _off(torch.full((sum(runs) + 2, H * D), 7.0, dtype=dtype, device=DEV), moved and out_off)
        w = torch.zeros(pages, G, 64, device=DEV)
        got = cache8.attention8(_off(q, moved and q_off), _on(codes), scales.to(DEV), _cu(runs), _i(held), table.to(DEV), 64, 0, 0.1, out, H, G, D, max(runs),
                                max(n + h for n, h in zip(runs, held)), weights=w)
        assert got is out and bool((out[-2:] == 7.0).all())
        seen.append((out.clone(), w))
    assert torch.equal(seen[0][0], seen[1][0]) and torch.equal(seen[0][1], seen[1][1])


# ---- scratch ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("with_weights", [False, True])
@pytest.mark.parametrize("shape", [(8, 2, 64), (16, 16, 128), (7, 1, 128)], ids=str)
@pytest.mark.parametrize("runs,held,window", [([64, 0, 50, 1], [6000, 5, 3000, 40], 100), ([200], [4999], 1), ([130, 70], [3, 6400], 64), ([300], [2000], 700)])
def test_a_windowed_prompt_expands_the_pages_it_sees(shape, runs, held, window, with_weights, monkeypatch):
    """Scratch for the window's pages of each sequence, not for all that its longest one holds; the result is held to the 64-bit one."""
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    H, G, D = shape
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64, windows=[max(0, h + 1 - window) for h in held])
    codes, scales = _cache(pages, G, 64, D, spread=1.0)
    q = (torch.randn(sum(runs), H, D) * 1.5).to(torch.bfloat16)
    scale, weights = 1.0 / math.sqrt(D) / 4, torch.rand(pages, G, 64)
    args = [q.to(DEV), _on(codes), scales.to(DEV), _cu(runs), _i(held), table.to(DEV)]
    out, w = torch.full((sum(runs), H * D), float("nan"), dtype=torch.bfloat16, device=DEV), weights.to(DEV) if with_weights else None
    longest = max(n + h for n, h in zip(runs, held))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    cache8.attention8(*args, 64, window, scale, out, H, G, D, max(runs), longest, weights=w)
    took = torch.cuda.max_memory_allocated() - before
    seen = len(runs) * ((max(runs) + window) // 64 + 2) * 2 * G * 64 * D * 2           # bfloat16 pages of what the sequences may see
    pieces = 4 * sum(runs) * H * (D + 1) * (longest // 512 + 2)
    assert took <= 1.01 * seen + pieces + (1 << 20), (took, seen, pieces)
    want, mags, units, p = plain.attention(q, codes, scales, runs, held, table, 64, window, scale, H, G, D)
    top = float((codes.view(torch.float8_e4m3fn).float().abs() * torch.pow(2.0, scales.float() - 127).repeat_interleave(16, -1)[..., None]).max())
    limit = _limit(torch.bfloat16, want, mags, units, D, longest, top)
    off = (out.cpu().double().view(want.shape) - want).abs()
    assert bool((off <= limit).all()), float((off / limit).max())
    if with_weights:
        want_w = weights.double()
        plain.add_weights(want_w, p, runs, held, table, 64, H, G)
        rel = float(2.02 * ((D + 8) * 4 * U * units).max()) + (longest + H // G * max(runs) + 16) * 4 * U
        assert bool(((w.cpu().double() - want_w).abs() <= rel * want_w.abs() + 1e-30).all())


# ---- plans for longer sequences than there are -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(16, 16, 128), (28, 4, 128), (8, 2, 64), (40, 2, 64), (3, 1, 256)], ids=str)
@pytest.mark.parametrize("longest", [1024, 8192, 40000])
@pytest.mark.parametrize("with_weights", [False, True])
def test_steps_planned_for_the_longest_sequence_there_could_be(dtype, shape, longest, with_weights):
    """As captured steps are: page tables and ranges for `longest` places, sequences that hold from none to some hundred, one that brings nothing."""
    from turboquant_cpp_b200.kernels import cache8
    (H, G, D), runs, held = shape, [1, 1, 0, 1, 1], [700, 0, 30, 63, 64]
    narrow, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    table = torch.full((len(runs), longest // 64), -1, dtype=torch.int32)
    table[:, :narrow.shape[1]] = narrow
    codes, scales = _cache(pages, G, 64, D)
    q, scale = (torch.randn(sum(runs), H, D) * 1.5).to(dtype), 1.0 / math.sqrt(D) / 4
    weights = torch.rand(pages, G, 64)
    out, w = torch.full((sum(runs), H * D), float("nan"), dtype=dtype, device=DEV), weights.to(DEV) if with_weights else None
    cache8.attention8(q.to(DEV), _on(codes), scales.to(DEV), _cu(runs), _i(held), table.to(DEV), 64, 0, scale, out, H, G, D, 1, longest, weights=w)
    want, mags, units, p = plain.attention(q, codes, scales, runs, held, narrow, 64, 0, scale, H, G, D)
    top = float((codes.view(torch.float8_e4m3fn).float().abs() * torch.pow(2.0, scales.float() - 127).repeat_interleave(16, -1)[..., None]).max())
    limit = _limit(dtype, want, mags, units, D, max(held) + 1, top)
    off = (out.cpu().double().view(want.shape) - want).abs()
    assert bool((off <= limit).all()), float((off / limit).max())
    if with_weights:
        want_w = weights.double()
        plain.add_weights(want_w, p, runs, held, narrow, 64, H, G)
        rel = float(2.02 * ((D + 8) * 4 * U * units).max()) + (max(held) + 1 + H // G + 16) * 4 * U
        assert bool(((w.cpu().double() - want_w).abs() <= rel * want_w.abs() + 1e-30).all())


# ---- scales and queries out of the ordinary ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs,held", [([1, 1], [200, 30]), ([60, 3], [100, 500])])
@pytest.mark.parametrize("scale", [-0.05, 0.0, 1e-30])
def test_scales_of_any_sign(dtype, runs, held, scale, monkeypatch):
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    H, G, D = 8, 2, 64
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D, spread=1.0)
    q, weights = torch.randn(sum(runs), H, D).to(dtype), torch.rand(pages, G, 64)
    want, mags, units, p = plain.attention(q, codes, scales, runs, held, table, 64, 0, scale, H, G, D)
    want_w = weights.double()
    plain.add_weights(want_w, p, runs, held, table, 64, H, G)
    got, got_w = _attend(q, codes, scales, runs, held, table, 64, 0, scale, H, G, D, weights)
    places = max(n + h for n, h in zip(runs, held))
    top = float((codes.view(torch.float8_e4m3fn).float().abs() * torch.pow(2.0, scales.float() - 127).repeat_interleave(16, -1)[..., None]).max())
    limit = _limit(dtype, want, mags, units, D, places, top)
    assert bool(((got.double().view(want.shape) - want).abs() <= limit).all())
    rel = float(2.02 * ((D + 8) * 4 * U * units).max()) + (places + H // G * max(runs) + 16) * 4 * U
    assert bool(((got_w.double() - want_w).abs() <= rel * want_w.abs() + 1e-30).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs,held", [([1, 1], [200, 30]), ([60, 3], [100, 500])])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite_is_its_rows_and_heads_alone(dtype, runs, held, bad, monkeypatch):
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    H, G, D = 8, 2, 64
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D, spread=1.0)
    q = torch.randn(sum(runs), H, D).to(dtype)
    want, _ = _attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D)
    q[0, 3, 7] = bad
    got, _ = _attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D)
    want, got = want.view(-1, H, D), got.view(-1, H, D)
    others = torch.ones(want.shape[:2], dtype=torch.bool)
    others[0, 3] = False
    assert torch.equal(got[others], want[others])
    assert math.isinf(bad) or bool(torch.isnan(got[0, 3]).all())


# ---- pools of more than 2^32 codes -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("runs,held", [([1, 1], [300, 64]), ([70, 3], [300, 64])])
def test_pages_behind_the_first_four_gigabytes(runs, held, monkeypatch):
    """A pool of 4.7 GB: sequences on its last pages get the bits they get on a small one's; its first pages stay as they are."""
    from turboquant_cpp_b200.kernels import cache8
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    H, G, D, budget = 16, 16, 128, 100
    T, rows = sum(runs), [n + h for n, h in zip(runs, held)]
    table, pages = _pages(rows, 64, spare=4)
    new = torch.tensor([p for p in range(pages) if p not in table.flatten().tolist()], dtype=torch.int32)[:4].view(2, 2)
    codes, scales = _cache(pages, G, 64, D, spread=1.0)
    qkv, w0 = torch.randn(T, (H + 2 * G) * D).to(torch.bfloat16).to(DEV), torch.rand(pages, G, 64)
    seen = []
    for before in (0, 18000):
        c, s, w = cache8.storage(before + pages, G, 64, D, DEV, weights=True)
        c[before:].view(torch.uint8).copy_(codes)
        s[before:].copy_(scales)
        w[before:].copy_(w0)
        on = lambda t: torch.where(t >= 0, t + before, t).to(torch.int32).to(DEV)
        q, out = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV), torch.empty(T, H * D, dtype=torch.bfloat16, device=DEV)
        cu, h = _cu(runs), _i(held)
        cache8.write_rows8(qkv, None, None, None, "half", torch.zeros(T, dtype=torch.int32, device=DEV), cu, h, on(table), 64, q, c, s, H, G, D, max(runs))
        cache8.attention8(q, c, s, cu, h, on(table), 64, 0, 0.08, out, H, G, D, max(runs), max(rows), weights=w)
        kept = cache8.evict8(c, s, w, _i(rows), on(table), on(new), 64, budget, 8)
        seen.append([t.clone() for t in (q, out, c[before:].view(torch.uint8), s[before:], w[before:], kept)])
        assert not bool(w[:before].any()) and not bool(c[:before].view(torch.uint8).any()) and bool((s[:before] == 1).all())
        del c, s, w
    for a, b in zip(*seen):
        assert torch.equal(a, b)
