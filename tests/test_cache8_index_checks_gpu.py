"""The index checks of the 8-bit cache's kernels (builds with TQ_DEBUG_INDEX=1): a page or a column that is not there is recorded, valid memory is used
instead, the kernel runs to its end, and the host raises when it looks.  In a process of its own, which launches nothing with a bad index unless the
library says that it is a checked build."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = r'''
import ctypes, os, sys
import numpy as np, torch
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))
import turboquant_cpp_b200 as tq
from turboquant_cpp_b200.csrc import build
from turboquant_cpp_b200.kernels import cache8

assert build.DEBUG_INDEX, "this process was to load the checked builds"
DEV = "cuda:0"
i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)
for name in ("cache8", "attention8", "evict", "prompt8", "attention_prefill"):
    rec = (ctypes.c_int * 4)()
    assert build.load_kernel(name).tq_index_fault_read(rec) == 1, f"{name} is not a checked build"

H, G, D, PAGE, PAGES = 4, 2, 64, 64, 8
codes, scales, weights = cache8.storage(PAGES, G, PAGE, D, DEV, weights=True)
codes.view(torch.uint8).copy_(torch.randint(0, 100, codes.shape, dtype=torch.uint8))
scales.fill_(120)


def after(fn):
    fn()
    torch.cuda.synchronize()                  # the kernels ran to their ends
    return build.index_faults()


def bad(found, library, what):
    assert any(f.startswith(library + ":") and what in f for f in found), (library, what, found)


def write(table, runs, held):
    T = sum(runs)
    cache8.write_rows8(torch.randn(T, (H + 2 * G) * D, device=DEV), None, None, None, "half", i32(np.zeros(T)), i32(np.concatenate([[0], np.cumsum(runs)])), i32(held),
                       i32(table), PAGE, torch.empty(T, H, D, device=DEV), codes, scales, H, G, D, max(runs))


def attend(table, runs, held, longest, window=0, sums=True, dtype=torch.bfloat16):
    T = sum(runs)
    q, out = torch.randn(T, H, D, device=DEV).to(dtype), torch.empty(T, H * D, dtype=dtype, device=DEV)
    cache8.attention8(q, codes, scales, i32(np.concatenate([[0], np.cumsum(runs)])), i32(held), i32(table), PAGE, window, 0.1, out, H, G, D, max(runs), longest,
                      weights=weights if sums else None)


def evict(table, new, lengths, budget, recent=2):
    cache8.evict8(codes, scales, weights, i32(lengths), i32(table), i32(new), PAGE, budget, recent)


good = [[1, 2], [4, 3]]
# what is in order leaves no record: empty runs, pages given back behind a window, pages that short sequences do not have
assert after(lambda: write(good, [1, 3], [100, 0])) == []
for runs in ([1, 1], [60, 0], [9, 2]):
    assert after(lambda: attend(good, runs, [60, 62], 128)) == []
assert after(lambda: attend([[-1, 2], [4, -1]], [1, 1], [100, 30], 128, window=30)) == []
assert after(lambda: evict([[1, 2], [4, -1]], [[5, 6], [7, -1]], [100, 40], 65)) == []
assert after(lambda: evict([[1, 2]], [[5, -1]], [100], 64)) == []
# a page outside the cache, a page given back, a place beyond the table
for table, held, what in (([[1, 900], [4, 3]], [100, 0], "page id"), ([[1, 2], [-1, 3]], [100, 5], "page id"), (good, [200, 5], "position beyond")):
    for runs in ([1, 1], [3, 2]):
        bad(after(lambda: write(table, runs, held)), "cache8", what)
    for sums in (False, True):
        for dtype in (torch.bfloat16, torch.float32):
            for runs in ([1, 1], [3, 2]):
                bad(after(lambda: attend(table, runs, held, 256, sums=sums, dtype=dtype)), "attention8", what)
cache8.PROMPT_WORK = 0
bad(after(lambda: attend([[1, 900], [4, 3]], [50, 2], [70, 0], 128)), "prompt8", "page id")
bad(after(lambda: attend(good, [50, 2], [200, 0], 256)), "prompt8", "position beyond")
bad(after(lambda: evict([[1, 900]], [[5]], [100], 64)), "evict", "page id")
bad(after(lambda: evict([[1, 2]], [[800]], [100], 64)), "evict", "page id")
bad(after(lambda: evict([[1, 2]], [[800]], [20], 64)), "evict", "page id")
assert after(lambda: attend(good, [50, 2], [70, 0], 128)) == []       # the record was cleared
print("8-bit index checks ok")
'''


def test_checked_builds_record_bad_pages_and_go_on():
    r = subprocess.run([sys.executable, "-c", f"ROOT = {ROOT!r}\n" + SCRIPT], capture_output=True, text=True, timeout=900, env=dict(os.environ, TQ_DEBUG_INDEX="1"))
    assert r.returncode == 0 and "8-bit index checks ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
