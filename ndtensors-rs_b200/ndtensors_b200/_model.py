"""What the language-model operators share: element types, streams, checks.

A call for a few tokens costs the host more than the GPU, so the plain cases
go through ``calls``, a small C++ module (``csrc/torch_calls.cpp``) that
returns None for any other; the wrappers then check, lay out or refuse.  Where
that module is missing they make every call themselves, with the same results.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import warnings
from pathlib import Path

import torch
from torch.autograd import forward_ad

from ._lib import get_lib, last_error
from .tensor import NDTensorsError, StatusCode


class _NoCalls:
    """In place of the C++ module: no call is a plain one, so the Python functions make them all."""

    @staticmethod
    def _none(*_):
        return None

    embedding = torch_embedding = scaled_linear = torch_scaled_linear = _none


def _load_calls(path=Path(__file__).resolve().parent.parent / "lib" / "ndt_torch_calls.so"):
    lib = get_lib()
    names = ("scaled_linear_dev", "scaled_linear_fwd_dev", "scaled_linear_vjp_dev", "embedding_dev", "embedding_grad_dev", "last_error")
    try:
        loader = importlib.machinery.ExtensionFileLoader("ndt_torch_calls", str(path))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("ndt_torch_calls", loader))
        loader.exec_module(module)
    except ImportError as e:  # not built, or for another torch
        warnings.warn(f"{path.name} does not load, so small calls take longer on the host; build it with "
                      f"`make -C ndtensors-rs_b200` ({e})", RuntimeWarning, stacklevel=2)
        return _NoCalls()
    module.bind([ctypes.cast(getattr(lib, f"ndt_b200_{n}"), ctypes.c_void_p).value for n in names], NDTensorsError)
    return module


calls = _load_calls()

#: element type codes of the C ABI
REAL = {torch.float32: 2, torch.bfloat16: 3, torch.float16: 4}
FLOAT8 = {torch.float8_e4m3fn: 5, torch.float8_e5m2: 6}

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_entries: dict = {}


def launch(name: str, device: int, *args) -> None:
    """Call the C entry point with the device current, its current stream as the last argument; raise its error
    (ValueError for sizes that do not fit)."""
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = getattr(get_lib(), name)
    if device == _current_device():
        status = f(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = f(*args, _raw_stream(device))
    if status == 0:
        return
    if status == StatusCode.SHAPE_MISMATCH:
        raise ValueError(last_error())
    raise NDTensorsError(f"{last_error()} (status {status})")


def device_of(what: str, first, *others) -> int:
    """The CUDA device that every tensor given is on."""
    device = first.get_device()
    if device < 0:
        raise NDTensorsError(f"{what}: the tensors must be CUDA tensors (there is no CPU compute path)")
    for t in others:
        if t is not None and t.get_device() != device:
            raise NDTensorsError(f"{what}: the tensors must be on one device")
    return device


def no_gradient(what: str, instead: str, *tensors) -> None:
    """Refuse inputs that ask for a gradient: the result would carry none."""
    asked = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    if not asked and forward_ad._current_level >= 0:
        asked = any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    if asked:
        raise NDTensorsError(f"{what}: an input requires a gradient, and the result would carry none: {instead}")


def plain(*tensors):
    """The tensors with the numbers that they stand for in memory (torch may hold a tensor as its opposite)."""
    return [t if t is None or not t.is_neg() else t.resolve_neg() for t in tensors]


def out_of(what: str, out) -> None:
    """A result can be written to ``out`` as it lies."""
    if out is not None and out.is_neg():
        raise ValueError(f"{what}: out must not have torch's negative bit")


def written(out) -> None:
    """``out`` was changed in place: a graph that saved it before must not be differentiated with what it holds now."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def code_of(what: str, name: str, dtype, allowed) -> int:
    """The C ABI's code of an element type, one of those allowed."""
    code = allowed.get(dtype)
    if code is None:
        raise TypeError(f"{what}: {name} must be one of {', '.join(str(d)[6:] for d in allowed)}, got {str(dtype)[6:]}")
    return code


def rows_of(x):
    """x as a matrix of its last axis (a view where its strides allow)."""
    if x.dim() == 2:
        return x
    lead = 1
    for n in x.shape[:-1]:
        lead *= n
    return x.reshape(lead, x.shape[-1])


def unit_rows(x):
    """The matrix x with unit stride along its rows and rows that do not overlap, copied only where it has not."""
    rs, cs = x.stride()
    return x if cs == 1 and rs >= x.shape[1] else x.contiguous()


__all__ = ["calls", "REAL", "FLOAT8", "launch", "device_of", "no_gradient", "plain", "out_of", "written", "code_of", "rows_of", "unit_rows"]
