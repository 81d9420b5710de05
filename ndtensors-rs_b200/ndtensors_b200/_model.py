"""What the language-model operators share: element types, streams, checks."""

from __future__ import annotations

import contextlib

import torch

from ._lib import get_lib, last_error
from .tensor import NDTensorsError, StatusCode

#: element type codes of the C ABI
CODES = {torch.float32: 2, torch.bfloat16: 3, torch.float16: 4, torch.float8_e4m3fn: 5, torch.float8_e5m2: 6}
REAL = (torch.float32, torch.bfloat16, torch.float16)
FLOAT8 = (torch.float8_e4m3fn, torch.float8_e5m2)

_raw_stream = torch._C._cuda_getCurrentRawStream
_here = contextlib.nullcontext()


def call(name: str, *args) -> None:
    """Call a C entry point; raise its error (ValueError for sizes that do not fit)."""
    status = getattr(get_lib(), name)(*args)
    if status == 0:
        return
    if status == StatusCode.SHAPE_MISMATCH:
        raise ValueError(last_error())
    raise NDTensorsError(f"{last_error()} (status {status})")


def on(device):
    """The context in which `device` is current, and its current stream's handle."""
    index = device.index
    if index == torch.cuda.current_device():
        return _here, _raw_stream(index)
    return torch.cuda.device(index), _raw_stream(index)


def check_cuda(what: str, first, *others) -> None:
    """Every tensor given is a CUDA tensor of one device."""
    if not first.is_cuda:
        raise NDTensorsError(f"{what}: the tensors must be CUDA tensors (there is no CPU compute path)")
    for t in others:
        if t is not None and t.device != first.device:
            raise NDTensorsError(f"{what}: the tensors must be on one device")


def check_type(what: str, name: str, dtype, allowed) -> None:
    if dtype not in allowed:
        raise TypeError(f"{what}: {name} must be one of {', '.join(str(d)[6:] for d in allowed)}, got {str(dtype)[6:]}")


def rows_of(x):
    """x as a matrix of its last axis (a view where its strides allow)."""
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def unit_rows(x):
    """x with unit stride along its last axis and rows that do not overlap, copied only where it has not."""
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= x.shape[1]:
        return x
    return x.contiguous()


__all__ = ["CODES", "REAL", "FLOAT8", "call", "on", "check_cuda", "check_type", "rows_of", "unit_rows"]
