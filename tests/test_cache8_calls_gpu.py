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
