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
