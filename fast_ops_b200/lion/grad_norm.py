"""The 2-norm over the gradients of a whole model, on the device.

`grad_norm` is the plain call; `Lion(..., max_grad_norm=c)` makes the same one before its step and
hands the clipping factor to the step's kernel in device memory, so that the gradients are never
rewritten and nothing waits for the host.
"""
from __future__ import annotations

import ctypes
from array import array
from functools import lru_cache
from operator import attrgetter
from typing import Iterable, List, Optional, Tuple

import torch
from torch import Tensor

from .. import _lib


def is_dense(t: Tensor) -> bool:
    """True when the tensor's elements fill one gap-free block of memory in some order
    (the reference's `is_non_overlapping_and_dense`, fast_ops/lion/lion_update.cu:109-112)."""
    if t.is_contiguous() or t.numel() == 0:
        return True
    strides = sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1)
    expect = 1
    for st, sz in strides:
        if st != expect:
            return False
        expect *= sz
    return True


_dtype_of = attrgetter("dtype")
_CODES = {torch.float16: _lib.FO_F16, torch.bfloat16: _lib.FO_BF16, torch.float32: _lib.FO_F32}


@lru_cache(maxsize=64)
def _workspace_doubles(n: int) -> int:
    return int(_lib.load().fo_grad_norm_workspace(n))


def _c_array(ctype, code: str, values: list):
    """A ctypes array of `values`; `code` is the array module's name for the type, whose arrays are filled
    faster from eight elements on (75 pointers: 3 us instead of 18)."""
    n = len(values)
    return (ctype * n)(*values) if n < 8 else (ctype * n).from_buffer(array(code, values))


class GradList:
    """ctypes image of the gradients of one norm call.  Checks and pointers are gathered column by
    column, by C functions mapped over the list: at a few hundred tensors the attribute accesses are what the call
    costs the host (300 tensors: 168 us per call with comprehensions, 109 like this)."""

    def __init__(self, grads: List[Tensor]):
        if not grads:
            raise RuntimeError("grad_norm needs at least one tensor")
        n = len(grads)
        try:
            devices = list(map(Tensor.get_device, grads))
        except TypeError:
            raise RuntimeError("gradients must be tensors") from None
        if min(devices) < 0:
            raise RuntimeError("fast_ops_b200 grad_norm needs CUDA tensors (there is no CPU path)")
        if devices.count(devices[0]) != n:
            raise RuntimeError("all gradients must be on one device")
        codes = list(map(_CODES.get, map(_dtype_of, grads)))
        if None in codes:
            raise RuntimeError(f"unsupported dtype {grads[codes.index(None)].dtype}")
        if not all(list(map(Tensor.is_contiguous, grads))) and not all([is_dense(g) for g in grads]):
            raise RuntimeError("expected tensor to be contiguous")
        ptrs = list(map(Tensor.data_ptr, grads))  # a sparse tensor has none and raises RuntimeError
        self.n, self.device, self.device_index = n, grads[0].device, devices[0]
        self.ptrs = _c_array(ctypes.c_void_p, "Q", ptrs)
        self.numels = _c_array(ctypes.c_int64, "q", list(map(Tensor.numel, grads)))
        self.dtypes = _c_array(ctypes.c_int, "i", codes)
        self.doubles = _workspace_doubles(n)

    def launch(self, max_norm: float, sumsq: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """The norm, a 0-d tensor, and a buffer whose first float is the clipping factor; `sumsq`, if
        given, receives the sum of squares as a double.  All of it is allocated by the call, so that
        calls on different streams or in different graphs share nothing."""
        norm = torch.empty((), dtype=torch.float32, device=self.device)
        buffer = torch.empty(self.doubles + 1, dtype=torch.float64, device=self.device)
        coef = buffer.data_ptr()
        _lib.check(_lib.load().fo_grad_norm(
            self.ptrs, self.numels, self.dtypes, self.n, max_norm, coef + 8, None if sumsq is None else sumsq.data_ptr(),
            norm.data_ptr(), coef, self.device_index, _lib.current_stream_ptr(self.device_index)))
        return norm, buffer


def grad_norm(grads: Iterable[Tensor]) -> Tensor:
    """The 2-norm of all elements of `grads` together, a 0-d fp32 tensor on their device.

    The tensors may be fp16, bf16 and fp32, mixed as they come, of any size, each dense in memory and
    all on one CUDA device (violations raise RuntimeError, an empty list too).  The squares of eight fp32
    elements at a time are summed in fp32 where it holds them, everything else in double, in a fixed
    order: the same gradients give the same bits, and squares that leave the range of fp32 count.  A
    norm beyond fp32 is infinite, non-finite gradients give a non-finite norm.  Not differentiable.  The
    call does not wait for the device and may be captured into a CUDA graph.
    """
    if isinstance(grads, Tensor):
        grads = [grads]
    with torch.no_grad():
        return GradList(list(grads)).launch(float("inf"))[0]


def finish_norm(sumsq: Tensor, max_norm: float) -> Tuple[Tensor, Tensor]:
    """(norm, clipping factor) from a sum of squares (a double on the device)."""
    norm, coef = (torch.empty((), dtype=torch.float32, device=sumsq.device) for _ in range(2))
    _lib.check(_lib.load().fo_grad_norm_finish(sumsq.data_ptr(), max_norm, norm.data_ptr(), coef.data_ptr(),
                                               sumsq.device.index, _lib.current_stream_ptr(sumsq.device.index)))
    return norm, coef


def shard_sumsq(flat_g: Tensor, begin: int, end: int) -> Tensor:
    """Sum of squares of elements [begin, end) of a flat gradient buffer, a one-element double."""
    sumsq = torch.empty(1, dtype=torch.float64, device=flat_g.device)
    GradList([flat_g[begin:end]]).launch(float("inf"), sumsq)
    return sumsq
