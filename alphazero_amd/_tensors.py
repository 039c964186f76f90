"""What the operators that take torch tensors need to hand them to libnnb.so."""
from __future__ import annotations

import contextlib
import ctypes as C

import torch
import torch.autograd.forward_ad as forward_ad

from ._lib import NnbError

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # nnb_dtype


def dtype_code(t: torch.Tensor, name: str) -> int:
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} is {t.dtype}: expected float32, float16 or bfloat16")
    return DTYPES[t.dtype]


_STAY = contextlib.nullcontext()


def on_device(t):
    """Makes the tensor's GPU current, which the library launches on."""
    device = t.device
    if device.type != "cuda":
        raise NnbError(f"a tensor on {device}: the kernels run on an MI355X only (there is no CPU path)")
    # switching devices costs more than a small launch: only where it changes something
    return _STAY if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def stream_of(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(torch._C._cuda_getCurrentRawStream(t.get_device()))


def ptr(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


def no_grad(what: str, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NnbError(f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:
        no_tangent(what, *tensors)


def no_tangent(what: str, *tensors):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NnbError(f"{what} has no forward-mode derivative: call it on tensors without a tangent")


def resolved(t: torch.Tensor) -> torch.Tensor:
    """t as its memory holds it: the imaginary part of a conjugate is a view marked as negated, over numbers that are not."""
    return t.resolve_neg() if t.is_neg() else t


def writable(t: torch.Tensor, name: str):
    if t.is_neg():
        raise ValueError(f"{name} is a negated view: the kernels would write the numbers without the sign")


def _span(t: torch.Tensor) -> tuple:
    """First and last address + 1 of the elements (torch's strides are never negative)."""
    reach = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (reach + 1) * t.element_size()


def overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two of t's elements may share memory: from the smallest stride up, each has to step over all that the smaller
    ones reach."""
    if t.numel() == 0:
        return False
    reach = 0
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s <= reach:
            return True
        reach += (n - 1) * s
    return False


def share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may have elements in common.  Column ranges of one buffer that lie apart are recognised; of
    other interleaved views it is assumed."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    strides = [s * t.element_size() for t in (a, b) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1]
    if strides and a.stride(-1) == 1 and b.stride(-1) == 1:
        row = min(strides)
        if row > 0 and all(s % row == 0 for s in strides):
            gap = (b0 - a0) % row                        # from a's columns to b's, around the row
            if gap >= a.shape[-1] * a.element_size() and gap + b.shape[-1] * b.element_size() <= row:
                return False
    return True
