"""The operators of the 8-bit cache against plain implementations: codes bit for bit, attention and sums of weights in 64 bits.

How far attention may be off, row by row (u = 2^-24, the half step of float32):
  * a score is a sum of hd products; accumulated in float32 in any order, with the factors ahead of it and truncating adders, it is off
    by at most (hd + 8) 4u of the sum of its products' magnitudes, and a softmax weight by twice that (its own score's and the sum's),
    times e^that <= 1.01 for the scores here, beside (n + 16) 4u for the exponentials, the sum over n places and the joins;
  * weights are held as float32, or as numbers of 16 bits whose two parts are off by 2^-22 and 2^-25 of the largest weight, for float32
    rows, and rounded to 16 bits, 2^-8 (bfloat16, the coarser), for bfloat16 rows;
  * the result is rounded to its type."""
import math

import pytest
import torch

from plain import cache8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
# (query heads, key/value heads, head size)
SHAPES = [(4, 4, 16), (6, 2, 32), (5, 1, 48), (8, 2, 64), (4, 2, 80), (16, 16, 128), (28, 4, 128), (9, 1, 128), (2, 1, 256), (40, 2, 64)]
# (runs, held)
STEPS = [([1], [0]), ([1], [15]), ([1], [16]), ([1], [700]), ([1, 1, 1], [63, 64, 130]), ([3, 0, 1], [5, 40, 200]), ([17, 64, 1, 2], [0, 63, 31, 14]),
         ([50], [0]), ([48, 200], [0, 77]), ([130, 49], [300, 16])]


@pytest.fixture(params=["by size", "prompt kernel"])
def prompts(request, monkeypatch):
    """Small steps go to the kernel of single tokens and short runs: with the second value, to the prompt kernel whatever their size."""
    if request.param != "by size":
        from turboquant_cpp_b200.kernels import cache8
        monkeypatch.setattr(cache8, "PROMPT_WORK", 0)


def _i(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(rows, page_size, spare=3, windows=None):
    """A page table for sequences of so many rows and the pool's pages (some belong to nobody)."""
    need = [-(-r // page_size) for r in rows]
    order = torch.randperm(sum(need) + spare).tolist()
    table = torch.full((len(rows), max(1, max(need))), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        for j in range(windows[i] // page_size if windows else 0):
            table[i, j] = -1
    return table, sum(need) + spare


def _cache(pages, G, page_size, D, spread=3.0):
    x = torch.randn(pages, 2, G, page_size // 16, 16, D) * torch.exp(spread * torch.randn(pages, 2, G, page_size // 16, 1, 1) / 2)
    b = torch.tensor([plain.byte_of(float(v)) for v in x.abs().amax((-1, -2)).flatten()], dtype=torch.int32).view(x.shape[:4])
    codes = (x * torch.pow(2.0, (127 - b).double())[..., None, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.view(pages, 2, G, page_size, D), b.to(torch.uint8)


def _cu(runs):
    return _i([sum(runs[:i]) for i in range(len(runs) + 1)])


def _on(codes):
    return codes.to(DEV).view(torch.float8_e4m3fn)


def _attend(q, codes, scales, runs, held, table, page_size, window, scale, H, G, D, weights=None, out=None):
    from turboquant_cpp_b200.kernels import cache8
    out = torch.full((q.shape[0], H * D), float("nan"), dtype=q.dtype, device=DEV) if out is None else out
    w = None if weights is None else weights.to(DEV)
    cache8.attention8(q.to(DEV), _on(codes), scales.to(DEV), _cu(runs), _i(held), table.to(DEV), page_size, window, scale, out, H, G, D, max(runs),
                      max(n + h for n, h in zip(runs, held)), weights=w)
    return out.cpu(), None if w is None else w.cpu()


def _limit(dtype, want, mags, units, D, places, top):
    """How far each element may be off; top: the largest |value| of the cache."""
    score = (D + 8) * 4 * U * units[..., None]
    weight = 2.02 * score + (places + 16) * 4 * U + (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -8)
    return weight * mags + 2.0 ** -25 * top * (places if dtype == torch.float32 else 1) + torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + 1e-30


# ---- the writer ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_written_codes_are_those_of_the_formulas(shape, dtype, step):
    from turboquant_cpp_b200.kernels import cache8
    (H, G, D), (runs, held), page_size = shape, STEPS[step], (64, 16, 32)[step % 3]
    pairing, biased, turned = ("half", "interleaved")[step % 2], step % 3 != 1, step % 4 != 3
    table, pages = _pages([n + h for n, h in zip(runs, held)], page_size)
    codes, scales = _cache(pages, G, page_size, D)
    T = sum(runs)
    qkv = (torch.randn(T, (H + 2 * G) * D) * torch.exp(2 * torch.randn(T, 1))).to(dtype)      # rows of unequal size: bytes grow
    bias = torch.randn((H + 2 * G) * D).to((torch.bfloat16, dtype)[step % 2]) if biased else None
    angle = torch.rand(1000, D // 2) * 6.3
    cos, sin = (torch.cos(angle), torch.sin(angle)) if turned else (None, None)
    positions = torch.randint(0, 1000, (T,), dtype=torch.int32)
    want_codes, want_scales = codes.clone(), scales.clone()
    want_q = plain.write(qkv, bias, cos, sin, pairing, positions, runs, held, table, page_size, want_codes, want_scales, H, G, D)
    q = torch.full((T, H, D), float("nan"), dtype=dtype, device=DEV)
    dev = lambda t: None if t is None else t.to(DEV)
    got_codes, got_scales = _on(codes), scales.to(DEV)
    cache8.write_rows8(dev(qkv), dev(bias), dev(cos), dev(sin), pairing, dev(positions), _cu(runs), _i(held), dev(table), page_size, q, got_codes, got_scales,
                       H, G, D, max(runs))
    assert torch.equal(got_scales.cpu(), want_scales)
    assert torch.equal(got_codes.view(torch.uint8).cpu(), want_codes)          # the whole pool: nothing else is touched
    assert torch.equal(q.cpu(), want_q.to(dtype))


def test_values_at_the_ends_of_the_range_and_those_that_are_not_finite():
    from turboquant_cpp_b200.kernels import cache8
    H = G = 1
    D, page_size = 32, 64
    specials = [0.0, -0.0, 448.0, 449.0, 464.0, 1e-45, 1e-38, -3e38, 3.4e38, math.inf, -math.inf, math.nan, 2.0 ** -130, 2.0 ** -9, 1.0625, 1.1875]
    for first in range(16):
        rows = torch.zeros(16, 3 * D)
        for r in range(16):
            v = specials[(first + r) % 16] if r < 3 else 0.0
            rows[r, D:] = torch.randn(2 * D) * (0.0 if abs(v) < 1e-30 else 0.5)
            rows[r, D + r] = v
            rows[r, 2 * D + 3] = v
        table, pages = _pages([64], page_size)
        codes, scales = _cache(pages, G, page_size, D)
        want_codes, want_scales = codes.clone(), scales.clone()
        plain.write(rows, None, None, None, "half", None, [16], [0], table, page_size, want_codes, want_scales, H, G, D)
        got_codes, got_scales, q = _on(codes), scales.to(DEV), torch.empty(16, 1, D, device=DEV)
        cache8.write_rows8(rows.to(DEV), None, None, None, "half", torch.zeros(16, dtype=torch.int32, device=DEV), _cu([16]), _i([0]), table.to(DEV), page_size,
                           q, got_codes, got_scales, H, G, D, 16)
        assert torch.equal(got_scales.cpu(), want_scales), first
        assert torch.equal(got_codes.view(torch.uint8).cpu(), want_codes), first


def test_a_step_written_again_leaves_the_same_bits():
    """What a decode step that is launched ahead, dropped and run again relies on."""
    from turboquant_cpp_b200.kernels import cache8
    H, G, D, runs, held = 4, 2, 64, [1, 1, 20], [37, 64, 9]
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D)
    got_codes, got_scales = _on(codes), scales.to(DEV)
    qkv = (8 * torch.randn(22, (H + 2 * G) * D)).to(DEV)
    seen = []
    for _ in range(2):
        q = torch.empty(22, H, D, device=DEV)
        cache8.write_rows8(qkv, None, None, None, "half", torch.zeros(22, dtype=torch.int32, device=DEV), _cu(runs), _i(held), table.to(DEV), 64, q, got_codes,
                           got_scales, H, G, D, 20)
        seen.append((got_codes.view(torch.uint8).clone(), got_scales.clone()))
    assert torch.equal(seen[0][0], seen[1][0]) and torch.equal(seen[0][1], seen[1][1])


# ---- attention -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attention_and_sums_of_weights(shape, dtype, step, prompts):
    (H, G, D), (runs, held) = shape, STEPS[step]
    window = (0, 40, 0, 1, 0, 100)[(step + SHAPES.index(shape)) % 6]
    page_size = (64, 32, 64, 16)[step % 4]
    gone = [max(0, h + 1 - window) for h in held] if window else None          # pages no row sees are given back
    table, pages = _pages([n + h for n, h in zip(runs, held)], page_size, windows=gone)
    codes, scales = _cache(pages, G, page_size, D)
    q = (torch.randn(sum(runs), H, D) * 1.5).to(dtype)
    scale = 1.0 / math.sqrt(D) / 4
    weights = torch.rand(pages, G, page_size)
    want, mags, units, p = plain.attention(q, codes, scales, runs, held, table, page_size, window, scale, H, G, D)
    want_w = weights.double()
    plain.add_weights(want_w, p, runs, held, table, page_size, H, G)
    places = max(n + h for n, h in zip(runs, held))
    top = float((codes.view(torch.float8_e4m3fn).float().abs() * torch.pow(2.0, scales.float() - 127).repeat_interleave(16, -1)[..., None]).max())
    limit = _limit(dtype, want, mags, units, D, places, top)
    for with_weights in (False, True):
        got, got_w = _attend(q, codes, scales, runs, held, table, page_size, window, scale, H, G, D, weights if with_weights else None)
        off = (got.double().view(want.shape) - want).abs()
        assert bool((off <= limit).all()), (float((off / limit).max()), with_weights)
        if with_weights:
            # a weight is off by its score's error and that of the row's sum; then the sums over rows and heads, in float32
            rel = float(2.02 * ((D + 8) * 4 * U * units).max()) + (places + H // G * max(runs) + 16) * 4 * U
            off = (got_w.double() - want_w).abs()
            assert bool((off <= rel * want_w.abs() + 1e-30).all()), float((off / (rel * want_w.abs() + 1e-30)).max())


@pytest.mark.parametrize("runs,held", [([1, 1], [200, 30]), ([60, 1], [0, 100])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_lies_behind_a_row_does_not_reach_it(dtype, runs, held, prompts):
    """Codes and bytes behind the last row (of pages used before) are NaN or the largest there are; the result keeps its bits."""
    H, G, D = 8, 2, 128
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D)
    q = torch.randn(sum(runs), H, D).to(dtype)
    seen = []
    for fill, byte in ((0x7f, 254), (0x7e, 240), (0, 1)):
        for s, (n, h) in enumerate(zip(runs, held)):
            last = n + h
            page, row = int(table[s, (last - 1) // 64]), (last - 1) % 64 + 1
            codes[page, :, :, row:] = fill
            scales[page, :, :, -(-row // 16):] = byte
        others = [p for p in range(pages) if p not in table.flatten().tolist()]
        codes[others] = fill
        seen.append(_attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D, torch.zeros(pages, G, 64)))
    for out, w in seen:
        assert bool(torch.isfinite(out).all()) and torch.equal(out, seen[0][0]) and torch.equal(w, seen[0][1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs", [[1], [70]])
def test_a_value_that_is_not_finite_is_lost_where_it_is_seen(dtype, runs, prompts):
    H, G, D, held = 4, 2, 128, [90]
    table, pages = _pages([held[0] + runs[0]], 64)
    codes, scales = _cache(pages, G, 64, D)
    at = held[0] + runs[0] - 1                                       # the last row's value, one element, one head
    codes[int(table[0, at // 64]), 1, 1, at % 64, 5] = 0x7f
    q = torch.randn(sum(runs), H, D).to(dtype)
    got, _ = _attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D)
    lost = torch.isnan(got.view(-1, H, D))
    want = torch.zeros_like(lost)
    want[-1, 2:, 5] = True
    assert torch.equal(lost, want)
    codes[int(table[0, at // 64]), 0, 0, at % 64, 9] = 0x7f             # and its key, another head
    got, _ = _attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D)
    want[-1, :2] = True
    assert torch.equal(torch.isnan(got.view(-1, H, D)), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs", [[1], [70]])
def test_blocks_of_very_unequal_bytes(dtype, runs, prompts):
    """Values of 2^30 whose weight is next to nothing beside values of 1, and rows of queries up to 2^60 and down to 2^-60."""
    H, G, D, held = 2, 1, 64, [150]
    n = held[0] + runs[0]
    table, pages = _pages([n], 64)
    codes, scales = _cache(pages, G, 64, D, spread=0.0)
    scales[int(table[0, 0]), 1, 0, 1] += 30
    scales[int(table[0, 1]), 1, 0, 0] -= 60
    q = torch.randn(sum(runs), H, D)
    for size in (0.0, 60.0, -60.0):
        x = (q * 2.0 ** size).to(dtype)
        scale = 2.0 ** -size / math.sqrt(D)
        want, mags, units, _ = plain.attention(x, codes, scales, runs, held, table, 64, 0, scale, H, G, D)
        got, _ = _attend(x, codes, scales, runs, held, table, 64, 0, scale, H, G, D)
        limit = _limit(dtype, want, mags, units, D, n, 0.0) + 2.0 ** -25 * n * mags.amax(-1, keepdim=True)
        off = (got.double().view(want.shape) - want).abs()
        assert bool((off <= limit).all()), (size, float((off / limit).max()))


def test_rows_behind_the_last_sequence_stay_and_a_graph_replays():
    from turboquant_cpp_b200.kernels import cache8
    H, G, D, held = 16, 4, 128, [130, 70, 5]
    table, pages = _pages([h + 1 for h in held], 64)
    codes, scales = _cache(pages, G, 64, D)
    q = torch.randn(5, H, D).to(torch.bfloat16).to(DEV)                 # two rows belong to nobody
    out = torch.full((5, H * D), 7.0, dtype=torch.bfloat16, device=DEV)
    w0 = torch.rand(pages, G, 64, device=DEV)
    args = lambda o, w: (q, c, b, cu, h, t, 64, 0, 0.08, o, H, G, D, 1, 192, w)
    c, b, cu, h, t = _on(codes), scales.to(DEV), _cu([1, 1, 1]), _i(held), table.to(DEV)
    w = w0.clone()
    cache8.attention8(*args(out, w))
    assert bool((out[3:] == 7.0).all()) and bool((out[:3] != 7.0).any())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out2, w2 = torch.full_like(out, 7.0), w0.clone()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            cache8.attention8(*args(out2, w2))
        w2.copy_(w0)
        g.replay()
    side.synchronize()
    assert torch.equal(out, out2) and torch.equal(w, w2)


def test_sums_of_weights_are_the_same_bits_every_time(prompts):
    H, G, D, runs, held = 28, 4, 128, [1, 1, 90], [500, 63, 200]
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D)
    q = torch.randn(sum(runs), H, D).to(torch.bfloat16)
    seen = [_attend(q, codes, scales, runs, held, table, 64, 0, 0.08, H, G, D, torch.zeros(pages, G, 64)) for _ in range(5)]
    for out, w in seen:
        assert torch.equal(out, seen[0][0]) and torch.equal(w, seen[0][1])


# ---- eviction ----------------------------------------------------------------------------------------------------------
EVICTIONS = [([300, 64, 1], 64, 16), ([300, 299, 65], 64, 64), ([100, 17, 16, 15], 16, 0), ([2000], 1000, 100), ([5000, 40], 333, 7), ([70], 1, 0), ([70], 1, 1),
             ([33, 32], 32, 5), ([0, 90], 50, 20), ([1100], 1030, 3)]


@pytest.mark.parametrize("shape", [(1, 16), (2, 48), (4, 128), (3, 256)], ids=str)
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("case", range(len(EVICTIONS)))
def test_eviction_keeps_the_rows_it_should(shape, kind, case):
    from turboquant_cpp_b200.kernels import cache8
    (G, D), (lengths, budget, recent), page_size = shape, EVICTIONS[case], (64, 16)[case % 2]
    per = -(-budget // page_size)
    table, pages = _pages([max(1, n) for n in lengths], page_size, spare=3 + per * len(lengths))
    taken = set(table.flatten().tolist())
    free = [p for p in range(pages) if p not in taken]
    new_table = torch.tensor(free[:per * len(lengths)], dtype=torch.int32).view(len(lengths), per)
    codes, scales = _cache(pages, G, page_size, D, spread=6.0)
    w = torch.exp(3 * torch.randn(pages, G, page_size))
    if kind == "ties":
        w = torch.randint(0, 3, w.shape).float()
    if kind == "odd":
        pick = torch.randint(0, 8, w.shape)
        for i, v in enumerate([math.nan, -math.nan, 0.0, -0.0, -1.0, 1e-45, math.inf]):
            w[pick == i] = v
        codes[torch.rand(codes.shape) < 0.01] = 0x7f
    want_codes, want_scales, want_w = codes.clone(), scales.clone(), w.double()
    want = plain.evict(want_codes, want_scales, want_w, lengths, table, new_table, page_size, budget, recent)
    got_codes, got_scales, got_w = _on(codes), scales.to(DEV), w.to(DEV)
    kept = cache8.evict8(got_codes, got_scales, got_w, _i(lengths), table.to(DEV), new_table.to(DEV), page_size, budget, recent)
    assert torch.equal(kept.cpu(), want)
    assert torch.equal(got_scales.cpu(), want_scales)
    assert torch.equal(got_codes.view(torch.uint8).cpu(), want_codes)
    assert torch.equal(torch.nan_to_num(got_w.cpu().double(), nan=-7.0), torch.nan_to_num(want_w, nan=-7.0))


@pytest.mark.parametrize("lengths,budget,recent", [([60000, 3000, 49300], 5000, 70), ([1023, 1024, 1025, 1100], 900, 0), ([4100, 8200, 2049], 1900, 130)])
@pytest.mark.parametrize("close", [0, 3, 63, 64, 65, 900])
@pytest.mark.parametrize("page_size", [48, 64])
def test_rows_whose_weights_lie_close_together(lengths, budget, recent, close, page_size):
    """`close` rows around the last that stays differ in the lowest bits alone, or not at all; sequences of more rows than a block keeps among them."""
    from turboquant_cpp_b200.kernels import cache8
    G, D = 2, 16
    per = -(-budget // page_size)
    table, pages = _pages(lengths, page_size, spare=per * len(lengths))
    taken = set(table.flatten().tolist())
    new_table = torch.tensor([p for p in range(pages) if p not in taken], dtype=torch.int32).view(len(lengths), per)
    codes, scales = torch.zeros(pages, 2, G, page_size, D, dtype=torch.uint8), torch.full((pages, 2, G, page_size // 16), 127, dtype=torch.uint8)
    w = torch.zeros(pages, G, page_size)
    want = torch.full((len(lengths), G, budget), -1, dtype=torch.int32)
    want_w = torch.zeros(len(lengths), G, budget)
    for s, n in enumerate(lengths):
        places = torch.arange(n)
        for g in range(G):
            mine = torch.exp(4 * torch.randn(n)).clamp(1e-30, 1e30)
            rest, keep = max(0, n - recent), budget - recent
            if close and n > budget and rest > close:
                order = torch.randperm(rest)
                above = max(0, keep - (close + 1) // 2)                   # rows above the close ones
                mine[order[:above]] = 4.0 + mine[order[:above]]
                mine[order[above:above + close]] = 1.0 + torch.randint(0, 2 * close, (min(close, rest - above),)).float() * 2.0 ** -23
                mine[order[above + close:]] = 0.9 / (1.0 + mine[order[above + close:]])
            w[table[s, places // page_size].long(), g, places % page_size] = mine
            kept = plain.kept_places(mine.tolist(), budget, recent)
            want[s, g, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            want_w[s, g, :len(kept)] = mine[kept]
    got_w = w.to(DEV)
    kept = cache8.evict8(_on(codes), scales.to(DEV), got_w, _i(lengths), table.to(DEV), new_table.to(DEV), page_size, budget, recent)
    assert torch.equal(kept.cpu(), want)
    moved = got_w.cpu()[new_table.long()].transpose(1, 2).reshape(len(lengths), G, -1)[:, :, :budget]
    assert torch.equal(torch.where(want >= 0, moved, 0.0), want_w)


def test_eviction_refuses_weights_that_are_not_aligned():
    from turboquant_cpp_b200.kernels import cache8
    from turboquant_cpp_b200.kernels._call import KernelError
    codes, scales = cache8.storage(4, 1, 16, 16, DEV)[:2]
    weights = torch.zeros(4 * 16 + 1, device=DEV)[1:].view(4, 1, 16)
    with pytest.raises(KernelError, match="16-byte aligned"):
        cache8.evict8(codes, scales, weights, _i([20]), _i([0, 1]).view(1, 2), _i([2]).view(1, 1), 16, 16, 4)


# ---- together -----------------------------------------------------------------------------------------------------------
def test_a_sequence_from_its_prompt_through_evictions(prompts):
    """Write, attend with sums, evict, go on: every step against the plain forms on the plain forms' own cache."""
    from turboquant_cpp_b200.kernels import cache8
    H, G, D, page_size, budget, recent = 6, 2, 64, 64, 96, 16
    pool = 12
    codes, scales, weights = cache8.storage(pool, G, page_size, D, DEV, weights=True)
    pc, ps, pw = codes.view(torch.uint8).cpu(), scales.cpu(), weights.cpu().double()
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    held, position = 0, 0
    angle = torch.rand(1000, D // 2) * 6.3
    cos, sin = torch.cos(angle), torch.sin(angle)
    turn = 0
    for n in [200] + [1] * 3 + [30] + [1] * 40:
        qkv = torch.randn(n, (H + 2 * G) * D).to(torch.bfloat16)
        positions = torch.arange(position, position + n, dtype=torch.int32)
        q = torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV)
        cache8.write_rows8(qkv.to(DEV), None, cos.to(DEV), sin.to(DEV), "half", positions.to(DEV), _cu([n]), _i([held]), table.to(DEV), page_size, q, codes,
                           scales, H, G, D, n)
        plain.write(qkv, None, cos, sin, "half", positions, [n], [held], table, page_size, pc, ps, H, G, D)
        assert torch.equal(codes.view(torch.uint8).cpu(), pc) and torch.equal(scales.cpu(), ps)
        out = torch.empty(n, H * D, dtype=torch.bfloat16, device=DEV)
        cache8.attention8(q, codes, scales, _cu([n]), _i([held]), table.to(DEV), page_size, 0, 0.125, out, H, G, D, n, held + n, weights=weights)
        want, mags, units, p = plain.attention(q.cpu(), pc, ps, [n], [held], table, page_size, 0, 0.125, H, G, D)
        assert bool(((out.cpu().double().view(want.shape) - want).abs() <= _limit(torch.bfloat16, want, mags, units, D, held + n, 10.0)).all())
        plain.add_weights(pw, p, [n], [held], table, page_size, H, G)
        assert float((weights.cpu().double() - pw).abs().max()) < 1e-4 * float(pw.max())
        held += n
        position += n
        if held > budget + 16:
            free = [i for i in range(pool) if i not in table.flatten().tolist()][:2]
            new = torch.tensor([free], dtype=torch.int32)
            pw = weights.cpu().double()                     # the same sums on both sides: which of two nearly equal ones is larger is not the point
            kept = cache8.evict8(codes, scales, weights, _i([held]), table.to(DEV), new.to(DEV), page_size, budget, recent)
            assert torch.equal(kept.cpu(), plain.evict(pc, ps, pw, [held], table, new, page_size, budget, recent))
            table = torch.tensor([free + [i for i in range(pool) if i not in free][:2]], dtype=torch.int32)
            held = budget
            turn += 1
    assert turn >= 2


def test_a_small_scratch_takes_the_sequences_in_groups(monkeypatch):
    from turboquant_cpp_b200.kernels import cache8
    H, G, D, runs, held = 8, 2, 64, [60, 0, 33, 49, 1], [70, 9, 0, 200, 64]
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D)
    q = torch.randn(sum(runs), H, D).to(torch.bfloat16)
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    want, want_w = _attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D, torch.zeros(pages, G, 64))
    monkeypatch.setattr(cache8, "DENSE_BYTES", 2 * 2 * G * 64 * D * 2 * 4)          # two sequences of four pages
    got, got_w = _attend(q, codes, scales, runs, held, table, 64, 0, 0.1, H, G, D, torch.zeros(pages, G, 64))
    assert torch.equal(got, want) and torch.equal(got_w, want_w)


@pytest.mark.parametrize("shape", [(8, 2, 64), (16, 16, 128), (28, 4, 128), (9, 1, 128)], ids=str)
@pytest.mark.parametrize("runs,held,window", [([48], [3000], 0), ([300, 129, 0, 1], [900, 1500, 7, 2000], 0), ([200], [2500], 700), ([1000], [0], 0), ([60, 400], [1300, 13], 200)])
def test_prompts_whose_keys_are_cut_into_pieces(shape, runs, held, window, monkeypatch):
    """Few units of many keys: pieces joined by a second launch; held to what whole units are held to, the sums of weights among it."""
    from turboquant_cpp_b200.kernels import cache8
    H, G, D = shape
    # four or six pages a piece, whatever the rule says of these sizes; a walk may begin inside a piece's first page
    pages_of = 4 + 2 * (H % 8 == 0)
    monkeypatch.setattr(cache8, "PROMPT_WORK", 0)
    monkeypatch.setattr(cache8, "prefill_pieces", lambda *a: (-(-(max(n + h for n, h in zip(runs, held)) + 64) // (64 * pages_of)), pages_of))
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D, spread=1.0)
    q = (torch.randn(sum(runs), H, D) * 1.5).to(torch.bfloat16)
    scale = 1.0 / math.sqrt(D) / 4
    weights = torch.rand(pages, G, 64)
    want, mags, units, p = plain.attention(q, codes, scales, runs, held, table, 64, window, scale, H, G, D)
    want_w = weights.double()
    plain.add_weights(want_w, p, runs, held, table, 64, H, G)
    got, got_w = _attend(q, codes, scales, runs, held, table, 64, window, scale, H, G, D, weights)
    places = max(n + h for n, h in zip(runs, held))
    top = float((codes.view(torch.float8_e4m3fn).float().abs() * torch.pow(2.0, scales.float() - 127).repeat_interleave(16, -1)[..., None]).max())
    limit = _limit(torch.bfloat16, want, mags, units, D, places, top)
    off = (got.double().view(want.shape) - want).abs()
    assert bool((off <= limit).all()), float((off / limit).max())
    rel = float(2.02 * ((D + 8) * 4 * U * units).max()) + (places + H // G * max(runs) + 16) * 4 * U
    assert bool(((got_w.double() - want_w).abs() <= rel * want_w.abs() + 1e-30).all())


def test_calls_on_two_streams_at_once():
    """Each call's scratch is its own: steps of two caches on two streams give what they give one after the other."""
    from turboquant_cpp_b200.kernels import cache8
    H, G, D = 28, 4, 128
    jobs = []
    for runs, held in (([1] * 6, [900, 40, 333, 1500, 64, 2]), ([1, 1, 60], [3000, 16, 500])):
        table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
        codes, scales = _cache(pages, G, 64, D)
        q = torch.randn(sum(runs), H, D).to(torch.bfloat16).to(DEV)
        jobs.append([q, _on(codes), scales.to(DEV), _cu(runs), _i(held), table.to(DEV), max(runs), max(n + h for n, h in zip(runs, held)), torch.rand(pages, G, 64, device=DEV)])

    def call(job, out, w):
        q, codes, scales, cu, held, table, run, longest, _ = job
        cache8.attention8(q, codes, scales, cu, held, table, 64, 0, 0.08, out, H, G, D, run, longest, weights=w)
    want = []
    for job in jobs:
        out, w = torch.empty(job[0].shape[0], H * D, dtype=torch.bfloat16, device=DEV), job[8].clone()
        call(job, out, w)
        want.append((out, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[(torch.empty_like(out), job[8].clone()) for _ in range(20)] for (out, _), job in zip(want, jobs)]
    torch.cuda.synchronize()
    for i in range(20):
        for s, job, g in zip(streams, jobs, got):
            with torch.cuda.stream(s):
                call(job, *g[i])
    torch.cuda.synchronize()
    for (out, w), g in zip(want, got):
        for a, b in g:
            assert torch.equal(a, out) and torch.equal(b, w)


@pytest.mark.parametrize("runs,held", [([1, 1], [5, 64]), ([20, 3], [0, 33])])
def test_queries_alone(runs, held):
    """A layer that reads another layer's cache writes its queries and nothing else."""
    from turboquant_cpp_b200.kernels import cache8
    H, G, D = 6, 2, 32
    T = sum(runs)
    table, pages = _pages([n + h for n, h in zip(runs, held)], 64)
    codes, scales = _cache(pages, G, 64, D)
    qkv, bias = torch.randn(T, (H + 2 * G) * D, device=DEV).to(torch.bfloat16), torch.randn((H + 2 * G) * D, device=DEV)
    angle = torch.rand(300, D // 2, device=DEV) * 6.3
    positions = torch.randint(0, 300, (T,), dtype=torch.int32, device=DEV)
    both = []
    for c, s in ((_on(codes), scales.to(DEV)), (None, None)):
        q = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
        cache8.write_rows8(qkv, bias, torch.cos(angle), torch.sin(angle), "half", positions, _cu(runs), _i(held), table.to(DEV), 64, q, c, s, H, G, D, max(runs))
        both.append(q)
    assert torch.equal(*both)
    with pytest.raises(Exception):
        cache8.write_rows8(qkv, bias, None, None, "half", positions, _cu(runs), _i(held), table.to(DEV), 64, both[0], None, scales.to(DEV), H, G, D, max(runs))


@pytest.mark.parametrize("shape", [(28, 4, 128), (16, 16, 128), (8, 2, 64), (4, 2, 80), (3, 1, 256), (5, 1, 48)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairing,biased", [("half", True), ("interleaved", False), ("half", None)])
def test_long_prompts_are_written_as_their_pieces_are(shape, dtype, pairing, biased):
    """One step of long prompts, whose threads go through several heads, leaves the bits that steps of 48 rows leave: they end where a block does."""
    from turboquant_cpp_b200.kernels import cache8
    H, G, D = shape
    runs, held, page_size = [1600, 3, 1, 700, 0, 33, 16, 900], [21, 0, 15, 16, 7, 31, 64, 5], 32
    table, pages = _pages([n + h for n, h in zip(runs, held)], page_size)
    codes, scales = _cache(pages, G, page_size, D)
    T = sum(runs)
    qkv = torch.randn(T, (H + 2 * G) * D, device=DEV) * torch.exp(2 * torch.randn(T, 1, device=DEV))
    for value in (math.inf, -math.inf, math.nan):
        qkv.view(-1)[torch.randint(0, qkv.numel(), (400,), device=DEV)] = value
    qkv = qkv.to(dtype)
    bias = None if biased is None else torch.randn((H + 2 * G) * D, device=DEV).to(torch.bfloat16 if biased else dtype)
    angle = torch.rand(1000, D // 2, device=DEV) * 6.3
    cos, sin = torch.cos(angle), torch.sin(angle)
    positions = torch.randint(0, 1000, (T,), dtype=torch.int32, device=DEV)
    dev_table = table.to(DEV)

    def write(rows, runs, held, codes, scales, q):
        cache8.write_rows8(qkv[rows].contiguous(), bias, cos, sin, pairing, positions[rows].contiguous(), _cu(runs), _i(held), dev_table, page_size, q, codes, scales,
                           H, G, D, max(runs))

    everything = torch.arange(T, device=DEV)
    got_q, got_codes, got_scales = torch.empty(T, H, D, dtype=dtype, device=DEV), _on(codes), scales.to(DEV)
    write(everything, runs, held, got_codes, got_scales, got_q)
    alone = torch.empty_like(got_q)
    write(everything, runs, held, None, None, alone)
    want_q, want_codes, want_scales = torch.empty_like(got_q), _on(codes), scales.to(DEV)
    starts, done = [sum(runs[:i]) for i in range(len(runs))], [0] * len(runs)
    while done != runs:
        now = [min(n - d, 48 - (h + d) % 16) for n, d, h in zip(runs, done, held)]
        rows = torch.tensor([s + d + i for s, d, n in zip(starts, done, now) for i in range(n)], device=DEV)
        q = torch.empty(len(rows), H, D, dtype=dtype, device=DEV)
        write(rows, now, [h + d for h, d in zip(held, done)], want_codes, want_scales, q)
        want_q[rows] = q
        done = [d + n for d, n in zip(done, now)]
    assert torch.equal(got_scales, want_scales)
    assert torch.equal(got_codes.view(torch.uint8), want_codes.view(torch.uint8))
    bits = torch.int16 if dtype == torch.bfloat16 else torch.int32
    assert torch.equal(got_q.view(bits), want_q.view(bits)) and torch.equal(alone.view(bits), want_q.view(bits))
