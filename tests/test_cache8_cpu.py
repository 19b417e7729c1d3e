"""What the 8-bit cache's entry points refuse, before anything is launched (no GPU), and the plain forms' own arithmetic."""
import math

import pytest
import torch

from plain import cache8_plain as plain

from turboquant_cpp_b200.kernels import KernelError, cache8

H, G, D, PAGE = 4, 2, 32, 64


def _i(values):
    return torch.tensor(values, dtype=torch.int32)


def _state(**other):
    codes, scales, weights = cache8.storage(3, G, PAGE, D, "cpu", weights=True)
    s = dict(codes=codes, scales=scales, weights=weights, table=_i([[0, 1]]), cu=_i([0, 2]), held=_i([5]), qkv=torch.zeros(2, (H + 2 * G) * D),
             q=torch.zeros(2, H, D), out=torch.zeros(2, H * D), cos=torch.zeros(9, D // 2), sin=torch.zeros(9, D // 2), bias=None, positions=_i([5, 6]),
             new_table=_i([[2]]), lengths=_i([70]), budget=32, recent=4, page=PAGE, hd=D, window=0)
    s.update(other)
    return s


def _write(s):
    cache8.write_rows8(s["qkv"], s["bias"], s["cos"], s["sin"], "half", s["positions"], s["cu"], s["held"], s["table"], s["page"], s["q"], s["codes"], s["scales"],
                       H, G, s["hd"], 2)


def _attend(s):
    cache8.attention8(s["q"], s["codes"], s["scales"], s["cu"], s["held"], s["table"], s["page"], s["window"], 0.1, s["out"], H, G, s["hd"], 2, 7, weights=s["weights"])


def _evict(s):
    cache8.evict8(s["codes"], s["scales"], s["weights"], s["lengths"], s["table"], s["new_table"], s["page"], s["budget"], s["recent"])


BAD_CACHE = [dict(codes=torch.zeros(3, 2, G, PAGE, D)), dict(codes=torch.zeros(3, 2, G, 48, D, dtype=torch.uint8).view(torch.float8_e4m3fn)),
             dict(scales=torch.zeros(3, 2, G, 4)), dict(scales=torch.zeros(3, 2, G, 8, dtype=torch.uint8)), dict(table=_i([0, 1])),
             dict(table=torch.zeros(1, 2, dtype=torch.int64))]


@pytest.mark.parametrize("call", [_write, _attend, _evict])
@pytest.mark.parametrize("bad", range(len(BAD_CACHE)))
def test_a_cache_of_other_shapes_is_refused(call, bad):
    with pytest.raises(KernelError):
        call(_state(**BAD_CACHE[bad]))


@pytest.mark.parametrize("bad", [dict(cu=_i([0, 1, 2])), dict(held=_i([5, 5])), dict(held=torch.tensor([5])), dict(cu=torch.tensor([0, 2])), dict(positions=_i([5])),
                                 dict(positions=torch.tensor([5, 6])), dict(q=torch.zeros(2, H, D, dtype=torch.bfloat16)), dict(q=torch.zeros(1, H, D)), dict(sin=None),
                                 dict(cos=torch.zeros(9, D)), dict(cos=torch.zeros(9, D // 2, dtype=torch.float64)), dict(bias=torch.zeros(D)),
                                 dict(qkv=torch.zeros(2, (H + G) * D))])
def test_steps_that_do_not_fit_are_not_written(bad):
    with pytest.raises(KernelError):
        _write(_state(**bad))


@pytest.mark.parametrize("bad", [dict(cu=_i([0, 1, 2])), dict(held=_i([5, 5])), dict(held=torch.tensor([5])), dict(out=torch.zeros(2, H * D, dtype=torch.bfloat16)),
                                 dict(out=torch.zeros(2, D)), dict(q=torch.zeros(2, H, 16)), dict(weights=torch.zeros(3, G, PAGE, dtype=torch.float64)),
                                 dict(weights=torch.zeros(3, H, PAGE))])
def test_steps_that_do_not_fit_are_not_attended(bad):
    with pytest.raises(KernelError):
        _attend(_state(**bad))


@pytest.mark.parametrize("bad", [dict(lengths=_i([70, 70])), dict(lengths=torch.tensor([70])), dict(new_table=_i([2])), dict(new_table=_i([[2], [1]])), dict(budget=65),
                                 dict(budget=0, recent=0), dict(recent=33), dict(recent=-1), dict(new_table=torch.tensor([[2]]))])
def test_evictions_that_do_not_fit_are_refused(bad):
    with pytest.raises(KernelError):
        _evict(_state(**bad))


@pytest.mark.parametrize("heads", [(4, 3), (0, 2), (4, 0)])
def test_heads_that_do_not_divide(heads):
    codes, scales, _ = cache8.storage(3, heads[1], PAGE, D, "cpu")
    s = _state()
    with pytest.raises(KernelError):
        cache8.attention8(torch.zeros(2, heads[0], D), codes, scales, s["cu"], s["held"], s["table"], PAGE, 0, 0.1, torch.zeros(2, heads[0] * D), *heads, D, 2, 7)
    with pytest.raises(KernelError):
        cache8.write_rows8(torch.zeros(2, (heads[0] + 2 * heads[1]) * D), None, None, None, "half", s["positions"], s["cu"], s["held"], s["table"], PAGE,
                           torch.zeros(2, heads[0], D), codes, scales, *heads, D, 2)


@pytest.mark.parametrize("call", [_write, _attend, _evict])
def test_there_is_no_cpu_path(call):
    with pytest.raises(KernelError):
        call(_state())


@pytest.mark.parametrize("page_size,head_dim", [(64, 24), (64, 272), (64, 0), (8, 64), (40, 64)])
def test_sizes_the_cache_does_not_take(page_size, head_dim):
    with pytest.raises(KernelError):
        cache8.storage(2, 1, page_size, head_dim, "cpu")


@pytest.mark.parametrize("top,b", [(0.0, 1), (448.0, 127), (448.5, 128), (896.0, 128), (1.0, 119), (3.4e38, 247), (1e-45, 1), (2.0 ** -126 * 448, 1), (2.0 ** -125 * 448, 2)])
def test_the_byte_is_the_smallest_that_holds_the_largest_magnitude(top, b):
    top = float(torch.tensor(top))
    assert plain.byte_of(top) == b
    assert top <= 448 * 2.0 ** (b - 127) and (b == 1 or top > 448 * 2.0 ** (b - 128))


def test_plain_codes_round_to_the_nearest():
    x = torch.linspace(-448, 448, 4001)
    got = plain.encode(x, 127).view(torch.float8_e4m3fn).double()
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    best = (x.double()[:, None] - every).abs().amin(1)
    assert torch.equal((x.double() - got).abs(), best)
    assert plain.encode(torch.tensor([math.inf, -math.inf, math.nan]), 127).tolist() == [0x7f] * 3


def test_plain_choice_of_rows():
    nan = math.nan
    assert plain.kept_places([1.0, 3.0, 2.0, 0.0], 2, 1) == [1, 3]
    assert plain.kept_places([1.0, 1.0, 1.0, 0.0], 3, 1) == [0, 1, 3]
    assert plain.kept_places([nan, 0.0, nan, -1.0], 2, 0) == [1, 3]
    assert plain.kept_places([5.0, 1.0], 4, 1) == [0, 1]


def test_declared_arguments_are_those_of_the_sources():
    """A letter per argument: an address, a whole number or a float, as the entry points are written."""
    import os
    import re

    from conftest import ROOT
    csrc = os.path.join(ROOT, "turboquant.cpp_b200", "csrc")
    text = "".join(open(os.path.join(csrc, f), encoding="utf-8").read() for f in ("cache8.cu", "attention8.cu", "prompt8.cu", "evict.cu", "attention_prefill.cu"))
    found = dict(re.findall(r"TQ_EXPORT int (tq_\w+)\((.*?)\)\s*\{", text, re.S))
    assert set(found) - {"tq_attention_prefill_dense"} == set(cache8._SIGNATURES) | set(cache8._PACKED)
    kind = lambda a: "p" if "*" in a or "cudaStream_t" in a else "f" if a.split()[0] == "float" else "i"
    for name, signature in cache8._SIGNATURES.items():
        assert "".join(kind(a.strip()) for a in found[name].split(",")) == signature, name
    for name, layout in cache8._PACKED.items():
        struct = re.search(r"c8_call<(\w+)>", text[text.index(f"TQ_EXPORT int {name}("):]).group(1)
        members = re.search(r"struct " + struct + r" \{(.*?)\};", text, re.S).group(1)
        kinds = "".join(kind(line) * (line.count(",") + 1) for line in (x.strip() for x in members.split(";")) if line)
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Pif])", layout))
        assert kinds.replace("p", "P") == want, name


def test_ranges_fill_the_device_and_no_more():
    r = cache8.ranges_for
    assert r(1024, 128, 592) == 1 and r(592, 2000, 592) == 1                # as many tiles as there is room for, or more
    assert r(1, 3, 592) == 1                                              # a few keys: one turn of one CTA's warps
    for tiles, blocks in ((16, 44), (32, 2031), (4, 8000), (128, 256), (600, 128)):
        n = r(tiles, blocks, 592)
        assert 1 < n <= min(64, blocks // 4) and (tiles > 592 or tiles * n <= 592)


def test_prompt_units_are_cut_where_few_of_them_are_long():
    from turboquant_cpp_b200.kernels.attention import prefill_pieces
    cut = lambda *a: prefill_pieces(*a, 148)
    assert cut(12000, 8, 2667, 2667, 16, 16, 128, 0) == (1, 0)             # more units than the device takes at once
    assert cut(2048, 1, 2048, 2048, 16, 16, 128, 0) == (1, 0)              # nearly as many
    assert cut(500, 1, 500, 500, 16, 16, 128, 0) == (1, 0)                 # few keys
    assert cut(1000, 2, 667, 9668, 28, 4, 128, 4096) == (1, 0)
    for args in ((500, 1, 500, 3500, 16, 16, 128, 0), (60, 1, 60, 5000, 28, 4, 128, 0), (64, 4, 16, 40000, 16, 16, 64, 0), (200, 1, 200, 9000, 8, 2, 64, 4096)):
        pieces, pages = cut(*args)
        keys = args[3] if not args[7] else args[7] + 256
        assert pieces > 1 and pages % 2 == 0 and pages >= 8 and pieces * pages * 64 >= keys + 127
        units = args[1] * args[4] * -(-args[2] // 256)
        assert pieces * units <= 2 * 148
    assert cut(1 << 20, 1, 256, 1 << 30, 1, 1, 128, 0) == (1, 0)           # more scratch than a step may take
