"""Glue between torch tensors and the C launchers of the kernel libraries."""
from __future__ import annotations

import ctypes
import struct
from operator import index
from typing import List, Optional

import torch

from ..csrc.build import load_kernel

F32, BF16 = 0, 1


class KernelError(RuntimeError):
    """A launcher refused its arguments or the launch failed; the message is the launcher's."""


def code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return F32
    if dtype == torch.bfloat16:
        return BF16
    raise KernelError(f"kernels take float32 or bfloat16 tensors, got {dtype}")


def ptr(t: Optional[torch.Tensor]) -> Optional[ctypes.c_void_p]:
    if t is None:
        return None
    if not t.is_cuda:
        raise KernelError("kernels take CUDA tensors; there is no CPU path")
    if not t.is_contiguous():
        raise KernelError("kernels take contiguous tensors")
    return ctypes.c_void_p(t.data_ptr())


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)


def stream() -> ctypes.c_void_p:
    """The current stream of the current device as the launchers take it.  Every launch asks, so this goes to
    torch's C entry points where this build of torch has them (a tenth of the cost of building a Stream object)."""
    if _raw_stream is not None and _raw_device is not None:
        return ctypes.c_void_p(_raw_stream(_raw_device()))
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


LAUNCHES = 0     # kernels of this library launched so far (counted by the wrappers)


def check(lib_name: str, rc: int, kernels: int = 1) -> None:
    global LAUNCHES
    LAUNCHES += kernels
    if rc != 0:
        lib = load_kernel(lib_name)
        raise KernelError(lib.tq_last_error().decode("utf-8", "replace") or f"{lib_name}: error {rc}")


def declared(lib: ctypes.CDLL, name: str, signature: str):
    """A launcher of a loaded kernel library with its argument types declared, which is cheaper to call than one that gets ctypes objects:
    signature has a letter per argument, p for an address (an int or None), i for a whole number, f for a float."""
    kinds = {"p": ctypes.c_void_p, "i": ctypes.c_int, "f": ctypes.c_float}
    fn = getattr(lib, name)
    fn.argtypes = [kinds[c] for c in signature]
    return fn


def packed(lib: ctypes.CDLL, name: str, layout: str):
    """A launcher of a loaded kernel library that takes one packed struct, as a function of the struct's members: `layout` in the letters of the
    struct module, addresses first (P), then whole numbers (i), then floats (f).  The launcher gets the bytes, padded at their end as C pads
    the struct, and how many they are, which it checks.  Four times as fast as as many declared arguments."""
    fn = getattr(lib, name)
    fn.argtypes = [ctypes.c_char_p, ctypes.c_int]
    call = struct.Struct("@" + layout + "0P")
    pack, size = call.pack, call.size
    return lambda *members: fn(pack(*members), size)


def addresses(*tensors: Optional[torch.Tensor]) -> List[int]:
    """What `ptr` gives, as plain ints (0 for None) for launchers with declared or packed arguments, and behind them the current stream.  Launches go to the current
    device: tensors of another GPU are refused instead of read from there."""
    if not tensors[0].is_cuda:
        ptr(tensors[0])                     # raises
    here = _raw_device() if _raw_device is not None else torch.cuda.current_device()
    out: List[int] = []
    for t in tensors:
        if t is None:
            out.append(0)
            continue
        if t.get_device() != here or not t.is_contiguous():
            ptr(t)                          # raises, unless the device is the wrong one
            raise KernelError(f"a tensor lies on GPU {t.get_device()}, the current device is {here}")
        out.append(t.data_ptr())
    out.append(_raw_stream(here) if _raw_stream is not None else torch.cuda.current_stream().cuda_stream)
    return out


def ints(*values) -> map:
    """Whole numbers of any integer type (numpy's among them) as the plain ints that ctypes passes on without a declaration."""
    return map(index, values)


def want_int32(t: torch.Tensor, what: str) -> None:
    if t.dtype != torch.int32:
        raise KernelError(f"{what} must be int32, got {t.dtype}")


def want_f32(t: torch.Tensor, what: str) -> None:
    if t.dtype != torch.float32:
        raise KernelError(f"{what} must be float32, got {t.dtype}")
