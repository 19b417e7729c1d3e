"""The 8-bit cache in plain torch on the CPU: rows to codes in float32 as the formulas say, attention and sums of weights in float64."""
import math

import torch

BLOCK = 16


def byte_of(top: float) -> int:
    """The smallest b >= 1 with top <= 448 * 2^(b - 127)."""
    if top == 0.0:
        return 1
    m, e = math.frexp(top)
    return max(1, e - 9 + (1 if m > 0.875 else 0) + 127)


def encode(x: torch.Tensor, b: int) -> torch.Tensor:
    """float32 values as the codes (uint8) of a block with byte b."""
    y = (x.double() * 2.0 ** (127 - b)).float()                       # a power of two: exact, or far below the smallest code
    return torch.where(torch.isfinite(x), y, torch.full_like(y, math.nan)).to(torch.float8_e4m3fn).view(torch.uint8)


def again(codes: torch.Tensor, shift: int) -> torch.Tensor:
    """Codes (uint8) rounded again after a factor of 2^-shift."""
    return (codes.view(torch.float8_e4m3fn).double() * 2.0 ** -shift).float().to(torch.float8_e4m3fn).view(torch.uint8)


def rotate(x, cos, sin, pairing):
    """x [T, heads, hd] float32; cos, sin [T, hd / 2]."""
    half = x.shape[-1] // 2
    u, v = (x[..., :half], x[..., half:]) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    c, s = cos[:, None], sin[:, None]
    a, b = u * c - v * s, u * s + v * c
    return torch.cat([a, b], -1) if pairing == "half" else torch.stack([a, b], -1).flatten(-2)


def write(qkv, bias, cos, sin, pairing, positions, runs, held, table, page_size, codes, scales, H, G, D):
    """Changes codes (uint8) and scales in place; returns the queries as float32 [T, H, D].  All on the CPU."""
    x = qkv.float()
    if bias is not None:
        x = x + bias.float()
    x = x.view(-1, H + 2 * G, D)
    if cos is not None:
        x = torch.cat([rotate(x[:, :H + G], cos[positions.long()], sin[positions.long()], pairing), x[:, H + G:]], 1)
    t0 = 0
    for s, (n, h) in enumerate(zip(runs, held)):
        for first in range(h // BLOCK * BLOCK, h + n, BLOCK):
            lo, hi = max(first, h), min(first + BLOCK, h + n)
            if hi <= lo:
                continue
            page, row, old = int(table[s, first // page_size]), first % page_size, lo - first
            for plane in range(2):
                for g in range(G):
                    rows = x[t0 + lo - h:t0 + hi - h, H + plane * G + g]
                    top = torch.where(torch.isfinite(rows), rows.abs(), torch.zeros_like(rows)).max()
                    was = int(scales[page, plane, g, row // BLOCK]) if old else 1
                    b = max(was, byte_of(float(top)))
                    scales[page, plane, g, row // BLOCK] = b
                    if old:
                        codes[page, plane, g, row:row + old] = again(codes[page, plane, g, row:row + old], b - was)
                    codes[page, plane, g, row + old:row + old + hi - lo] = encode(rows, b)
        t0 += n
    return x[:, :H]


def rows_of(codes, scales, table, s, n, page_size):
    """(keys, values) [G, n, D] float64 of a sequence's first n places."""
    pages = table[s, :-(-n // page_size)].long().clamp(min=0)
    x = codes[pages].view(torch.float8_e4m3fn).double() * torch.pow(2.0, scales[pages].double() - 127).repeat_interleave(BLOCK, -1)[..., None]
    x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
    return x[0], x[1]


def attention(q, codes, scales, runs, held, table, page_size, window, scale, H, G, D):
    """(out [T, H, D], the weighted sum of |values| [T, H, D], each row's largest possible score error in units of 2^-24 [T, H], the
    weights per sequence [H, n, places]) in float64."""
    out, mags, units, weights, t0 = [], [], [], [], 0
    for s, (n, h) in enumerate(zip(runs, held)):
        if n == 0:
            weights.append(None)
            continue
        k, v = rows_of(codes, scales, table, s, h + n, page_size)
        at, place = torch.arange(h, h + n)[:, None], torch.arange(h + n)[None]
        hidden = place > at
        if window:
            hidden = hidden | (at - place >= window)
        k, v = k.repeat_interleave(H // G, 0), v.repeat_interleave(H // G, 0)
        x = q[t0:t0 + n].double().view(n, H, D).transpose(0, 1)
        p = torch.softmax((x @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf), -1)
        seen = torch.zeros_like(p).masked_fill(~hidden, 1.0)
        # values in hidden places do not count, whatever they are
        zero = lambda t: torch.where(torch.isfinite(t), t, torch.zeros_like(t))
        o = p @ zero(v)
        bad = seen @ (~torch.isfinite(v)).double() > 0
        o = torch.where(bad, torch.full_like(o, math.nan), o)
        out.append(o.transpose(0, 1))
        mags.append((p @ zero(v).abs()).transpose(0, 1))
        units.append(((x.abs() @ zero(k).abs().transpose(1, 2) * abs(scale)).masked_fill(hidden, 0.0).amax(-1)).transpose(0, 1))
        weights.append(p)
        t0 += n
    return torch.cat(out), torch.cat(mags), torch.cat(units), weights


def add_weights(weights, p, runs, held, table, page_size, H, G):
    """weights [pages, G, page_size] float64, changed in place."""
    for s, (n, h) in enumerate(zip(runs, held)):
        if n == 0:
            continue
        j = torch.arange(h + n)
        page, row = table[s].long()[j // page_size], j % page_size
        got = p[s].view(G, H // G, n, h + n).sum((1, 2))                       # [G, places]
        was = torch.where(j < h, weights[page.clamp(min=0), :, row].T, torch.zeros_like(got))
        mine = page >= 0                                                       # given back: no row of the step sees it
        weights[page[mine], :, row[mine]] = (was + got).T[mine]


def kept_places(w, budget, recent):
    """The places that stay of a sequence whose rows have the sums w (a list of floats)."""
    n = len(w)
    if n <= budget:
        return list(range(n))
    rest = n - recent
    order = sorted(range(rest), key=lambda j: (-math.inf if math.isnan(w[j]) else w[j]), reverse=True)     # stable: the first of equal ones
    return sorted(order[:budget - recent]) + list(range(rest, n))


def evict(codes, scales, weights, lengths, table, new_table, page_size, budget, recent):
    """Changes codes (uint8), scales and weights in place; returns the places kept."""
    n, G = len(lengths), codes.shape[2]
    kept = torch.full((n, G, budget), -1, dtype=torch.int32)
    for s, length in enumerate(lengths):
        for g in range(G):
            w = [float(weights[int(table[s, j // page_size]), g, j % page_size]) for j in range(length)]
            mine = kept_places(w, budget, recent)
            kept[s, g, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            for first in range(0, len(mine), BLOCK):
                block = mine[first:first + BLOCK]
                page, row = int(new_table[s, first // page_size]), first % page_size
                for plane in range(2):
                    old = [int(scales[int(table[s, j // page_size]), plane, g, j % page_size // BLOCK]) for j in block]
                    for r, (j, b) in enumerate(zip(block, old)):
                        codes[page, plane, g, row + r] = again(codes[int(table[s, j // page_size]), plane, g, j % page_size], max(old) - b)
                    scales[page, plane, g, row // BLOCK] = max(old)
                for r, j in enumerate(block):
                    weights[page, g, row + r] = w[j]
    return kept
