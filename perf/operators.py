"""Attention over a cache of keys and values in 8 bits whose length stays bounded: the work whose speed is measured.

Four operators, as one layer of a model uses them on a step's tokens:

    write    bias and rotation on a step's fused projection; its queries to a buffer, its keys and values into the pages
    attend   causal attention of the step's queries over the pages (one token per sequence, or runs of many)
    weigh    the same, and the softmax weights that every cached row of a key/value head has received are added up
    evict    sequences that hold too many rows keep those with the largest sums, and the newest ones, on new pages

A cached element is an e4m3 code times 2^(b - 127), b one byte for 16 rows of a (page, plane, key/value head): the smallest
power of two under which the largest magnitude of the 16 rows is at most 448.  Rows that are already in a block when its
byte grows are rounded again.  What is not finite becomes NaN and leaves the byte alone.

codes [pages, 2 (keys, values), kv heads, 64, head size] e4m3; scales [pages, 2, kv heads, 4] uint8; weights [pages, kv heads,
64] float32.  Row t of sequence s lies at place held[s] + t - cu_seqlens[s], the place's page stands in the page table.
A pool's last page belongs to nobody.
"""
import math

import torch

own = False

PAGE, BLOCK, TOP = 64, 16, 448.0
DEVICE = "cuda:0"
POSITIONS = 40960                # rows of the rotation's tables
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------------------
# heads: query heads x key/value heads x head size; seqs: sequences of the step; new: tokens they bring together (absent:
# one each); held: rows the longest of them holds from before; gone: positions before its first row that were evicted
def listed():
    return [
        # one chat's next token, in the middle of a block of 16
        {"name": "write_1", "kind": "write", "heads": "16x16x128", "dtype": "bfloat16", "seqs": 1, "held": 700, "gone": 0, "bias": True, "pairing": "half"},
        # three prompts of unequal lengths in one step
        {"name": "write_prompts", "kind": "write", "heads": "16x16x128", "dtype": "bfloat16", "seqs": 3, "new": 4096, "held": 0, "gone": 0, "bias": True, "pairing": "half"},
        # one chat's next token
        {"name": "attend_1", "kind": "attend", "heads": "16x16x128", "dtype": "bfloat16", "seqs": 1, "held": 700, "window": 0},
        # a server's decode step
        {"name": "attend_64", "kind": "attend", "heads": "16x16x128", "dtype": "bfloat16", "seqs": 64, "held": 2048, "window": 0},
        # long documents, seven query heads on a key/value head
        {"name": "attend_long", "kind": "attend", "heads": "28x4x128", "dtype": "bfloat16", "seqs": 8, "held": 32500, "window": 0},
        # the 32-bit run that users compare with
        {"name": "attend_float32", "kind": "attend", "heads": "16x4x64", "dtype": "float32", "seqs": 8, "held": 2048, "window": 0},
        # eight whole prompts
        {"name": "attend_prompts", "kind": "attend", "heads": "16x16x128", "dtype": "bfloat16", "seqs": 8, "new": 12000, "held": 0, "window": 0},
        # pieces of prompts behind what their sequences hold already, inside a window
        {"name": "attend_pieces", "kind": "attend", "heads": "28x4x128", "dtype": "bfloat16", "seqs": 2, "new": 1000, "held": 9001, "window": 4096},
        # a decode step that adds up its weights
        {"name": "weigh_32", "kind": "weigh", "heads": "28x4x128", "dtype": "bfloat16", "seqs": 32, "held": 4096},
        # a prompt that does
        {"name": "weigh_prompt", "kind": "weigh", "heads": "16x16x128", "dtype": "bfloat16", "seqs": 1, "new": 2048, "held": 0},
        # one chat goes back to 1,024 rows
        {"name": "evict_1", "kind": "evict", "heads": "16x16x128", "seqs": 1, "held": 1088, "budget": 1024, "recent": 128},
        # a server's sequences after their prompts
        {"name": "evict_32", "kind": "evict", "heads": "28x4x128", "seqs": 32, "held": 7001, "budget": 2048, "recent": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "weigh", "weigh", "evict"])
    heads = rng.choice(["16x16x128", "16x16x128", "28x4x128", "28x4x128", "16x4x64", "6x2x32", "5x1x48", "8x2x256"])
    case = {"kind": kind, "heads": heads}
    H, G, D = (int(n) for n in heads.split("x"))
    if kind == "evict":
        held = _log(rng, 3, 16000)
        case.update(seqs=_log(rng, 1, max(1, min(48, 200000 // held))), held=held, budget=max(1, int(held * rng.uniform(0.2, 1.1))))
        return dict(case, recent=rng.randint(0, min(case["budget"], 512)))
    case["dtype"] = "float32" if rng.random() < 0.3 else "bfloat16"
    if rng.random() < 0.5:                        # one token per sequence
        held = _log(rng, 1, 30000)
        case.update(seqs=_log(rng, 1, max(1, min(64, 130000 // held))), held=held)
    else:                                         # runs
        most = 4096 if D in (64, 128) and case["dtype"] == "bfloat16" else 700
        new = _log(rng, 2, most)
        case.update(seqs=rng.randint(1, min(4, new)), new=new, held=rng.choice([0, 0, _log(rng, 1, 5000)]))
    if kind == "write":
        return dict(case, gone=rng.choice([0, 0, rng.randint(1, 3000)]), bias=rng.random() < 0.5, pairing=rng.choice(["half", "half", "interleaved"]))
    if kind == "attend":
        case["window"] = rng.choice([0, 0, 0, _log(rng, 8, 4096)])
    return case


def _sizes(case):
    return tuple(int(n) for n in case["heads"].split("x"))


def _lens(case):
    """(rows each sequence brings, rows it holds): unequal, from the case alone."""
    n, most = case["seqs"], case["held"]
    held = [max(0, most - (i * 37) % max(1, most // 3 + 1)) for i in range(n)]
    if case["kind"] == "evict":
        return [0] * n, [max(1, h) for h in held]
    if "new" not in case:
        return [1] * n, held
    runs = [1 + (i + 1) * (case["new"] - n) // (n * (n + 1) // 2) for i in range(n)]
    runs[-1] += case["new"] - sum(runs)
    return runs, held


# ---- inputs ------------------------------------------------------------------------------------------------------
def _exponent(top):
    """The byte b of blocks whose largest magnitude is `top` (float32): the smallest with top <= 448 * 2^(b - 127), at least 1."""
    m, e = torch.frexp(top)
    return torch.where(top > 0, e.int() - 9 + (m > 0.875).int(), torch.full_like(e, -126, dtype=torch.int32)).clamp(-126, 127) + 127


def _power(n):
    """2^n for whole n from -126 to 127 (below: 2^-126), exactly."""
    return (n.int().clamp(min=-126) + 127 << 23).view(torch.float32)


def _to_codes(x):
    return torch.where(torch.isfinite(x), x, torch.full_like(x, math.nan)).to(torch.float8_e4m3fn)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(gen, rows, extra=0):
    """A page table for sequences of so many rows, pages in no order; (table, pages taken)."""
    need = [-(-r // PAGE) for r in rows]
    order = torch.randperm(sum(need) + extra, generator=gen, device=DEVICE, dtype=torch.int64).int()
    table = torch.full((len(rows), max(1, max(need))), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, order, at


def _rows_of_a_model(gen, shape):
    """Keys and values as trained models have them: channels of unequal size, a few far larger than the rest."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    size = torch.exp(0.4 * torch.randn(shape[-1], generator=gen, device=DEVICE))
    size = torch.where(torch.rand(shape[-1], generator=gen, device=DEVICE) < 0.02, size * 6.0, size)
    return x * size


def prepare(case, seed):
    H, G, D = _sizes(case)
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) & 0x7FFFFFFF)
    runs, held = _lens(case)
    rows = [r + h for r, h in zip(runs, held)]
    spare = 0
    if case["kind"] == "evict":
        spare = len(rows) * -(-case["budget"] // PAGE)
    table, order, used = _tables(gen, rows, extra=spare)
    pages = int(order.numel()) + 1
    st = {"case": case, "table": table, "held": _ints(held), "scale": 1.0 / math.sqrt(D)}
    x = _rows_of_a_model(gen, (pages, 2, G, PAGE // BLOCK, BLOCK, D))
    b = _exponent(x.abs().amax((-1, -2)))
    st["scales"] = b.to(torch.uint8)
    st["codes"] = _to_codes(x * _power(127 - b)[..., None, None]).view(pages, 2, G, PAGE, D)
    del x
    if case["kind"] in ("weigh", "evict"):       # sums of weights: few large ones, many small ones, some that are equal
        w = torch.exp(2.0 * torch.randn((pages, G, PAGE), generator=gen, device=DEVICE) - 3.0)
        st["weights"] = torch.where(torch.rand(w.shape, generator=gen, device=DEVICE) < 0.1, torch.zeros_like(w), w)
    if case["kind"] == "evict":
        per = -(-case["budget"] // PAGE)
        st["new_table"] = order[used:].view(len(rows), per).contiguous()
        st["most"] = max(held)
        return st
    dtype = DTYPES[case["dtype"]]
    T, n = sum(runs), len(runs)
    cu = [0]
    for r in runs:
        cu.append(cu[-1] + r)
    st.update(cu=_ints(cu), longest=max(runs), most=max(rows),
              seq=torch.repeat_interleave(torch.arange(n, device=DEVICE), torch.tensor(runs, device=DEVICE)))
    if case["kind"] == "write":
        width = (H + 2 * G) * D
        st["qkv"] = _rows_of_a_model(gen, (T, width)).to(dtype)
        st["bias"] = torch.randn(width, generator=gen, device=DEVICE).to(dtype) if case["bias"] else None
        i = torch.arange(D // 2, dtype=torch.float64, device=DEVICE)
        angle = torch.arange(POSITIONS, dtype=torch.float64, device=DEVICE)[:, None] * torch.pow(torch.tensor(1e6, dtype=torch.float64, device=DEVICE), -2.0 * i / D)
        st["cos"], st["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        st["positions"] = (st["held"][st["seq"]] + torch.arange(T, device=DEVICE) - st["cu"][st["seq"]] + case["gone"]).int()
        st["out"] = torch.empty((T, H, D), dtype=dtype, device=DEVICE)
        return st
    st["q"] = torch.randn((T, H, D), generator=gen, device=DEVICE).to(dtype)
    st["out"] = torch.empty((T, H * D), dtype=dtype, device=DEVICE)
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    H, G, D = _sizes(case)
    kind = case["kind"]
    if own:
        from turboquant_cpp_b200.kernels import cache8
        if kind == "write":
            cache8.write_rows8(st["qkv"], st["bias"], st["cos"], st["sin"], case["pairing"], st["positions"], st["cu"], st["held"],
                               st["table"], PAGE, st["out"], st["codes"], st["scales"], H, G, D, st["longest"])
        elif kind == "evict":
            kept = cache8.evict8(st["codes"], st["scales"], st["weights"], st["held"], st["table"], st["new_table"], PAGE,
                                 case["budget"], case["recent"])
            return {"kept": kept, "codes": st["codes"], "scales": st["scales"], "weights": st["weights"]}
        else:
            cache8.attention8(st["q"], st["codes"], st["scales"], st["cu"], st["held"], st["table"], PAGE, case.get("window", 0),
                              st["scale"], st["out"], H, G, D, st["longest"], st["most"], weights=st.get("weights"))
    elif kind == "write":
        _plain_write(st, H, G, D, case["pairing"])
    elif kind == "evict":
        return {"kept": _plain_evict(st, G, D, case["budget"], case["recent"]), "codes": st["codes"], "scales": st["scales"], "weights": st["weights"]}
    else:
        _plain_attention(st, H, G, D, case.get("window", 0))
    if kind == "write":
        return {"q": st["out"], "codes": st["codes"], "scales": st["scales"]}
    return {"out": st["out"], "weights": st["weights"]} if kind == "weigh" else {"out": st["out"]}


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _at(table, seqs, places, spare):
    """(page, row of the page) of sequences' places; the page nobody has where the table has none."""
    column = (places // PAGE).clamp(0, table.shape[1] - 1)
    page = table[seqs, column].long()
    return torch.where((page >= 0) & (places // PAGE < table.shape[1]), page, torch.full_like(page, spare)), places % PAGE


def _plain_write(st, H, G, D, pairing):
    seq, cu, held, table = st["seq"], st["cu"].long(), st["held"].long(), st["table"]
    codes, scales = st["codes"].view(torch.uint8), st["scales"]
    T, spare = seq.shape[0], codes.shape[0] - 1
    x = st["qkv"].float()
    if st["bias"] is not None:
        x = x + st["bias"].float()
    x = x.view(T, H + 2 * G, D)
    cos, sin = st["cos"][st["positions"].long()][:, None], st["sin"][st["positions"].long()][:, None]
    turned = x[:, :H + G]
    u, v = (turned[..., :D // 2], turned[..., D // 2:]) if pairing == "half" else (turned[..., 0::2], turned[..., 1::2])
    a, b = u * cos - v * sin, u * sin + v * cos
    turned = torch.cat([a, b], -1) if pairing == "half" else torch.stack([a, b], -1).flatten(-2)
    st["out"].copy_(turned[:, :H])
    kv = torch.stack([turned[:, H:], x[:, H + G:]], 1)                       # [T, 2, G, D]
    place = held[seq] + torch.arange(T, device=x.device) - cu[seq]
    page, row = _at(table, seq, place, spare)
    block = page * (PAGE // BLOCK) + row // BLOCK
    by_block = scales.permute(0, 3, 1, 2).reshape(-1, 2, G).int()            # a copy
    fresh = held[seq] <= place // BLOCK * BLOCK
    before = torch.where(fresh[:, None, None], torch.ones_like(by_block[block]), by_block[block])
    need = _exponent(torch.where(torch.isfinite(kv), kv.abs(), torch.zeros_like(kv)).amax(-1))
    now = torch.zeros_like(by_block).index_reduce_(0, block, torch.maximum(need, before), "amax")
    # the rows a run's first block holds already
    first = held // BLOCK * BLOCK
    some = torch.arange(held.shape[0], device=x.device)
    old_place = first[:, None] + torch.arange(BLOCK, device=x.device)
    old_page, old_row = _at(table, some[:, None], old_place, spare)
    old_block = old_page[:, 0] * (PAGE // BLOCK) + old_row[:, 0] // BLOCK
    grown = (now[old_block] - by_block[old_block]).clamp(min=0)              # [B, 2, G]; blocks that take no row: 0
    mine = (old_place < held[:, None])[:, :, None, None, None]
    old = codes[old_page, :, :, old_row]                                     # [B, 16, 2, G, D]
    again = (old.view(torch.float8_e4m3fn).float() * _power(-grown)[:, None, :, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[old_page, :, :, old_row] = torch.where(mine, again, old)
    codes[page, :, :, row] = _to_codes(kv * _power(127 - now[block])[..., None]).view(torch.uint8)
    scales[page, :, :, row // BLOCK] = now[block].to(torch.uint8)


def _rows(st, G, D):
    """Keys and values of every sequence, [seqs, 2, G, places, D] float32."""
    table = st["table"].long()
    table = torch.where(table >= 0, table, torch.full_like(table, st["codes"].shape[0] - 1))
    x = st["codes"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float()                        # [B, W, 2, G, 64, D]
    size = _power(st["scales"][table].int() - 127)              # [B, W, 2, G, 4]
    x = x.view(*x.shape[:4], PAGE // BLOCK, BLOCK, D) * size[..., None, None]
    return x.permute(0, 2, 3, 1, 4, 5, 6).reshape(x.shape[0], 2, G, -1, D)


def _plain_attention(st, H, G, D, window):
    seq, cu, held = st["seq"], st["cu"].long(), st["held"].long()
    kv = _rows(st, G, D)
    B, S, R, T = kv.shape[0], kv.shape[3], st["longest"], seq.shape[0]
    run = cu[1:] - cu[:-1]
    r = torch.arange(R, device=kv.device)
    mine = r < run[:, None]                                                  # [B, R]
    q = st["q"].float()[(cu[:-1, None] + r).clamp(max=T - 1)].view(B, R, G, H // G, D)
    s = torch.einsum("brghd,bgsd->bghrs", q, kv[:, 0]) * st["scale"]
    place = torch.arange(S, device=kv.device)
    at = (held[:, None] + r)[..., None]                                      # [B, R, 1]
    seen = (place <= at) & mine[..., None]
    if window > 0:
        seen &= at - place < window
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    del s
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = torch.einsum("bghrs,bgsd->brghd", p, kv[:, 1]).reshape(B, R, H * D)
    st["out"].copy_(out[seq, torch.arange(T, device=kv.device) - cu[seq]])
    if "weights" in st:
        add = p.sum((2, 3))                                                  # [B, G, S]
        page, row = _at(st["table"], torch.arange(B, device=kv.device)[:, None], place[None].expand(B, S), st["codes"].shape[0] - 1)
        before = st["weights"][page, :, row]                                 # [B, S, G]
        after = torch.where((place >= held[:, None])[..., None], torch.zeros_like(before), before) + add.transpose(1, 2)
        st["weights"][page, :, row] = torch.where((place < (held + run)[:, None])[..., None], after, before)


def _plain_evict(st, G, D, budget, recent):
    held, table, weights, codes, scales = st["held"].long(), st["table"], st["weights"], st["codes"].view(torch.uint8), st["scales"]
    B, S, spare = held.shape[0], table.shape[1] * PAGE, codes.shape[0] - 1
    place = torch.arange(S, device=held.device)
    page, row = _at(table, torch.arange(B, device=held.device)[:, None], place[None].expand(B, S), spare)
    w = weights[page, :, row].transpose(1, 2)                                # [B, G, S]
    rank = torch.nan_to_num(w, nan=-2e38)
    length = held[:, None, None]
    rank = rank.masked_fill(place >= length - recent, math.inf).masked_fill(place >= length, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.sort(torch.where(best < length, best, torch.full_like(best, S)), dim=-1).values      # [B, G, n]
    if kept.shape[-1] < budget:
        kept = torch.cat([kept, kept.new_full((B, G, budget - kept.shape[-1]), S)], -1)
    there = kept < length
    n = -(-budget // BLOCK) * BLOCK
    from_ = torch.cat([kept, kept.new_full((B, G, n - budget), S)], -1)      # whole blocks of 16
    good = from_ < length
    b, g = torch.arange(B, device=held.device)[:, None, None], torch.arange(G, device=held.device)[None, :, None]
    old_page, old_row = _at(table, b, torch.where(good, from_, torch.zeros_like(from_)), spare)
    old = torch.where(good[..., None], scales[old_page, :, g, old_row // BLOCK].int(), 0)             # [B, G, n, 2]
    top = old.view(B, G, n // BLOCK, BLOCK, 2).amax(3)                                                # [B, G, n / 16, 2]
    shift = (old - top.repeat_interleave(BLOCK, 2))[..., None]
    new = (codes[old_page, :, g, old_row].view(torch.float8_e4m3fn).float() * _power(shift)).to(torch.float8_e4m3fn).view(torch.uint8)
    sums = weights[old_page, g, old_row]
    to = torch.arange(n, device=held.device)
    new_page, new_row = _at(st["new_table"], b, to[None, None].expand(B, 1, n), spare)
    new_page, new_row = new_page.expand(B, G, n), new_row.expand(B, G, n)
    new_page = torch.where(good, new_page, torch.full_like(new_page, spare))
    # rows that are not there go to the page nobody has, as what it holds
    codes[new_page, :, g, new_row] = torch.where(good[..., None, None], new, codes[new_page, :, g, new_row])
    weights[new_page, g, new_row] = torch.where(good, sums, weights[new_page, g, new_row])
    block_page, block = new_page[..., ::BLOCK], new_row[..., ::BLOCK] // BLOCK
    scales[block_page, :, g, block] = torch.where(good[..., ::BLOCK, None], top.to(torch.uint8), scales[block_page, :, g, block])
    return torch.where(there, kept, torch.full_like(kept, -1)).int()


# ---- the least a pass has to do ----------------------------------------------------------------------------------
def work(case):
    H, G, D = _sizes(case)
    runs, held = _lens(case)
    row = 2 * G * (D + 1.0 / BLOCK)                                          # bytes of a cached row, all heads
    if case["kind"] == "evict":
        keep = sum(min(h, case["budget"]) for h in held)
        return {"bytes": 4.0 * G * sum(held) + keep * (2.0 * row + 8.0 * G + 4.0 * G), "flops": 0.0}
    el, T = (4 if case["dtype"] == "float32" else 2), sum(runs)
    if case["kind"] == "write":
        return {"bytes": T * ((2.0 * H + 2.0 * G) * D * el + 4.0 * D + row), "flops": 6.0 * T * (H + G) * D}
    window = case.get("window", 0)
    pairs = sum(min(p + 1, window) if window else p + 1 for n, h in zip(runs, held) for p in range(h, h + n))
    seen = sum(n + (min(h, window - 1) if window else h) for n, h in zip(runs, held))
    more = 8.0 * G * seen if case["kind"] == "weigh" else 0.0
    return {"bytes": 2.0 * el * T * H * D + row * seen + more, "flops": 4.0 * H * D * pairs}


# ---- the same in 64 bits, a sequence at a time -------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    H, G, D = _sizes(case)
    runs, held = _lens(case)
    if case["kind"] == "evict":
        return _exact_evict(case, st, G, D, held)
    if case["kind"] == "write":
        return _exact_write(case, st, H, G, D, runs, held)
    return _exact_attention(case, st, H, G, D, runs, held)


def _rounded(y):
    """The nearest e4m3 value of each y, |y| <= 448 (ties to the even one)."""
    _, e = torch.frexp(y)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=y.device), (e.clamp(min=-5) - 4).double())
    return torch.round(y / step) * step


def _byte(top):
    """The exponent byte of a block whose largest magnitude is `top`."""
    b = 1
    while top > TOP * 2.0 ** (b - 127):
        b += 64 if top > TOP * 2.0 ** (b + 64 - 127) else 8 if top > TOP * 2.0 ** (b + 8 - 127) else 1
    return b


def _values(st, s, rows):
    """(keys, values) of a sequence's first `rows` places, [G, rows, D] float64."""
    n = -(-rows // PAGE)
    page = st["table"][s, :n].long()
    x = st["codes"].view(torch.uint8)[page].view(torch.float8_e4m3fn).double()
    size = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), st["scales"][page].double() - 127.0)
    x = x * size.repeat_interleave(BLOCK, -1)[..., None]
    x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :rows]
    return x[0], x[1]


def _exact_attention(case, st, H, G, D, runs, held):
    out, sums, t0 = [], None if "weights" not in st else st["weights"].double(), 0
    for s, (n, h) in enumerate(zip(runs, held)):
        k, v = _values(st, s, h + n)
        at = torch.arange(h, h + n, device=DEVICE)[:, None]
        place = torch.arange(h + n, device=DEVICE)[None]
        hidden = place > at
        if case.get("window", 0):
            hidden |= place <= at - case["window"]
        q = st["q"][t0:t0 + n].double().view(n, G, H // G, D)
        o = torch.empty((n, G, H // G, D), dtype=torch.float64, device=DEVICE)
        for g in range(G):
            got = torch.zeros(h + n, dtype=torch.float64, device=DEVICE)
            for j in range(H // G):
                a = torch.softmax((q[:, g, j] @ k[g].T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
                o[:, g, j] = a @ v[g]
                got += a.sum(0)
            if sums is not None:
                page = st["table"][s].long().repeat_interleave(PAGE)[:h + n]
                row = torch.arange(h + n, device=DEVICE) % PAGE
                sums[page, g, row] = torch.where(torch.arange(h + n, device=DEVICE) < h, sums[page, g, row], 0.0) + got
        out.append(o.view(n, H * D))
        t0 += n
    return {"out": torch.cat(out)} if sums is None else {"out": torch.cat(out), "weights": sums}


def _exact_write(case, st, H, G, D, runs, held):
    x = st["qkv"].double() + (0.0 if st["bias"] is None else st["bias"].double())
    x = x.view(-1, H + 2 * G, D)
    pos = st["positions"].long()
    turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None]
    pair = x[:, :H + G].unflatten(-1, (2, D // 2)).transpose(-1, -2) if case["pairing"] == "half" else x[:, :H + G].unflatten(-1, (D // 2, 2))
    turned = torch.view_as_real(torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * turn)
    turned = (turned.transpose(-1, -2) if case["pairing"] == "half" else turned).flatten(-2)
    kv = torch.stack([turned[:, H:], x[:, H + G:]], 1).cpu()
    codes, scales, table = st["codes"].cpu().double(), st["scales"].cpu().int(), st["table"].cpu()
    t0 = 0
    for s, (n, h) in enumerate(zip(runs, held)):
        for first in range(h // BLOCK * BLOCK, h + n, BLOCK):
            page, row, old = int(table[s, first // PAGE]), first % PAGE, max(0, h - first)
            rows = kv[t0 + first + old - h:t0 + min(first + BLOCK, h + n) - h]
            top = rows.abs().amax((0, 3))
            for c in range(2):
                for g in range(G):
                    was = int(scales[page, c, g, row // BLOCK]) if old else 1
                    b = max(was, _byte(float(top[c, g])))
                    scales[page, c, g, row // BLOCK] = b
                    if b > was and old:
                        codes[page, c, g, row:row + old] = _rounded(codes[page, c, g, row:row + old] * 2.0 ** (was - b))
                    codes[page, c, g, row + old:row + old + rows.shape[0]] = _rounded(rows[:, c, g] * 2.0 ** (127 - b))
        t0 += n
    return {"q": turned[:, :H].contiguous(), "codes": codes, "scales": scales.to(torch.uint8)}


def _exact_evict(case, st, G, D, held):
    codes, scales, weights = st["codes"].cpu().double(), st["scales"].cpu().int(), st["weights"].cpu().double()
    table, new = st["table"].cpu().long(), st["new_table"].cpu().long()
    budget, recent = case["budget"], case["recent"]
    kept = torch.full((len(held), G, budget), -1, dtype=torch.int32)
    for s, h in enumerate(held):
        place = torch.arange(h)
        page, row = table[s].repeat_interleave(PAGE)[:h], place % PAGE
        n = min(h, budget)
        for g in range(G):
            if h <= budget:
                mine = place
            else:
                old = weights[page[:h - recent], g, row[:h - recent]]
                order = sorted(range(h - recent), key=(-old).tolist().__getitem__)[:budget - recent]
                mine = torch.tensor(sorted(order) + list(range(h - recent, h)), dtype=torch.int64)
            kept[s, g, :n] = mine.int()
            to = torch.arange(n)
            to_page, to_row = new[s].repeat_interleave(PAGE)[:n], to % PAGE
            weights[to_page, g, to_row] = weights[page[mine], g, row[mine]]
            for c in range(2):
                b = scales[page[mine], c, g, row[mine] // BLOCK]
                top = torch.zeros(-(-n // BLOCK), dtype=torch.int32).index_reduce_(0, to // BLOCK, b, "amax")
                size = torch.pow(torch.tensor(2.0, dtype=torch.float64), (b - top[to // BLOCK]).double())
                codes[to_page, c, g, to_row] = _rounded(codes[page[mine], c, g, row[mine]] * size[:, None])
                scales[to_page[::BLOCK], c, g, to_row[::BLOCK] // BLOCK] = top
    return {"kept": kept, "codes": codes, "scales": scales.to(torch.uint8), "weights": weights}
