"""Calls of the 8-bit cache's entry points that must end in an error, or stay within their bounds, before anything reaches the device (no GPU)."""
import ctypes

import pytest
import torch

from turboquant_cpp_b200.kernels import KernelError, cache8

H, G, D, PAGE = 4, 2, 32, 64


def _i(values):
    return torch.tensor(values, dtype=torch.int32)


# ---- eviction without sums of weights ------------------------------------------------------------------------------------
def test_eviction_without_weights_is_refused(monkeypatch):
    """Sums of weights are what rows are chosen by: a cache that keeps none cannot be evicted from.  The launcher is replaced by one that must not be reached."""
    def reached(*members):
        raise AssertionError("the launcher was called")
    monkeypatch.setattr(cache8, "_evict", lambda name: reached)
    monkeypatch.setattr(cache8, "addresses", lambda *tensors: [0 if t is None else t.data_ptr() for t in tensors] + [0])
    codes, scales, none = cache8.storage(3, G, PAGE, D, "cpu")
    assert none is None
    with pytest.raises(KernelError, match="weights"):
        cache8.evict8(codes, scales, none, _i([70]), _i([[0, 1]]), _i([[2]]), PAGE, 32, 4)


def test_the_launcher_refuses_an_eviction_without_weights():
    """Its own check, ahead of any launch: every other argument is one it would take."""
    evict = cache8._evict("tq_evict8")
    assert evict(16, 16, 0, 16, 16, 16, 16, 0, 2, 1, PAGE, 3, 1, G, D, 32, 4) != 0
    from turboquant_cpp_b200.csrc.build import load_kernel
    assert b"weights" in load_kernel("evict").tq_last_error()


# ---- packed calls ----------------------------------------------------------------------------------------------------------
def _c_struct(name):
    """The struct an entry point takes, from its source, as ctypes lays it out (C's rules: padding behind the last member too)."""
    import os
    import re

    from conftest import ROOT
    csrc = os.path.join(ROOT, "turboquant.cpp_b200", "csrc")
    text = "".join(open(os.path.join(csrc, f), encoding="utf-8").read() for f in ("cache8.cu", "attention8.cu", "evict.cu"))
    struct = re.search(r"c8_call<(\w+)>", text[text.index(f"TQ_EXPORT int {name}("):]).group(1)
    fields = []
    for line in (x.strip() for x in re.search(r"struct " + struct + r" \{(.*?)\};", text, re.S).group(1).split(";")):
        kind = ctypes.c_void_p if "*" in line or "cudaStream_t" in line else ctypes.c_float if line.startswith("float") else ctypes.c_int
        fields += [(f"m{len(fields) + i}", kind) for i in range(line.count(",") + 1)] if line else []
    return type(struct, (ctypes.Structure,), {"_fields_": fields})


@pytest.mark.parametrize("name", sorted(cache8._PACKED))
def test_a_packed_call_has_all_the_bytes_its_launcher_copies(name):
    from turboquant_cpp_b200.kernels import _call
    struct, seen = _c_struct(name), []

    class Fn:
        def __call__(self, data, *size):
            seen.append((data, size))
            return 0
    lib = type("Lib", (), {name: Fn()})()
    members = list(range(1, len(struct._fields_) + 1))
    assert _call.packed(lib, name, cache8._PACKED[name])(*members) == 0
    data, size = seen[0]
    assert len(data) == ctypes.sizeof(struct) and size == (len(data),)
    got = struct.from_buffer_copy(data)
    assert [getattr(got, f) for f, _ in struct._fields_] == members


@pytest.mark.parametrize("library,name", [("cache8", "tq_write8"), ("attention8", "tq_attention8"), ("evict", "tq_evict8")])
def test_a_packed_call_of_another_length_is_refused(library, name):
    """A layout that no longer is the launcher's: refused before a byte is read."""
    from turboquant_cpp_b200.csrc.build import load_kernel
    lib, size = load_kernel(library), ctypes.sizeof(_c_struct(name))
    fn = getattr(lib, name)
    was, fn.argtypes = fn.argtypes, [ctypes.c_char_p, ctypes.c_int]
    try:
        assert fn(bytes(size), size) == 0                                   # no sequences: nothing to do
        for other in (0, size - 4, size + 8):
            assert fn(bytes(size), other) != 0 and b"bytes" in lib.tq_last_error()
    finally:
        fn.argtypes = was


# ---- pages whose offsets would not fit ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("library,name", [("cache8", "tq_write8"), ("attention8", "tq_attention8"), ("evict", "tq_evict8")])
@pytest.mark.parametrize("page_size,nkv,hd,fits", [(1 << 17, 128, 128, False), (1 << 17, 64, 256, False), (1 << 17, 127, 128, True)])
def test_a_plane_of_a_page_stays_below_two_to_the_31_codes(library, name, page_size, nkv, hd, fits):
    """Offsets within a page are 32 bits wide.  (A page that fits is refused for its codes' alignment, the check behind it: nothing is launched.)"""
    from turboquant_cpp_b200.csrc.build import load_kernel
    lib, struct = load_kernel(library), _c_struct(name)
    order = {"tq_write8": [0, 0, 0, 1, page_size, 1, 1, 1, nkv, nkv, hd], "tq_attention8": [0, 1, page_size, 0, 1, 0, 16, 1, 1, 1, nkv, nkv, hd],
             "tq_evict8": [1, 1, page_size, 1, 1, nkv, hd, 16, 4]}[name]
    call = cache8._PACKED[name]
    addresses = [8] * int(call[:call.index("P")])
    members = addresses + order + ([0.1] if call.endswith("f") else [])
    assert len(members) == len(struct._fields_)
    assert getattr(cache8, f"_{library}")(name)(*members) != 0
    message = lib.tq_last_error()
    assert (b"codes a plane" in message) == (not fits) and (b"aligned" in message) == fits, message


# ---- options --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("options", [dict(cache_recent=16), dict(cache_dtype="e4m3", cache_recent=16), dict(cache_recent=-1), dict(cache_dtype="e4m3", cache_recent=1)])
def test_newest_rows_without_a_budget_are_refused(options):
    """`cache_recent` says how many of a budget's rows are the newest: without a budget it would do nothing."""
    import turboquant_cpp_b200 as tq
    from conftest import TINY_A
    for make in (lambda m: tq.Model.from_model(m, **options), lambda m: tq.Engine(m, max_tokens=64, **options)):
        with pytest.raises(ValueError, match="cache"):
            make(tq.build_model(TINY_A, "bfloat16"))


# ---- what the kernel ahead wrote ----------------------------------------------------------------------------------------------------
def test_data_of_the_kernel_ahead_is_not_read_as_read_only():
    """A kernel launched early may be resident while the kernel ahead still writes the queries, the codes and their bytes: for its lifetime they are not
    read-only, which __ldg would claim.  (Queries come as `const __restrict__` parameters: those are renewed behind the wait.)"""
    import os
    import re

    from conftest import ROOT
    csrc = os.path.join(ROOT, "turboquant.cpp_b200", "csrc")
    for name in ("cache8.cu", "cache8.cuh", "attention8.cu", "prompt8.cu", "evict.cu"):
        text = open(os.path.join(csrc, name), encoding="utf-8").read()
        assert not re.search(r"__ldg\s*\(", text), name
        for m in re.finditer(r"__restrict__ q,[^{]*\{(.*?)\n\}\n", text, re.S):
            assert "q = tq_fresh(q);" in m.group(1) or "tq_grid_wait()" not in m.group(1), (name, m.group(0)[:120])
