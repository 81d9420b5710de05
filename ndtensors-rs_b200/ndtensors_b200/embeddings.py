"""Embedding lookup with scaling, and its gradient: contraction with a one-hot
tensor that is never formed.  Everything runs on torch's current stream."""

from __future__ import annotations

import torch
from torch.autograd import Function

from ._model import CODES, REAL, call, check_cuda, check_type, on, unit_rows


def _check_ids(what: str, ids) -> None:
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: ids must be int32 or int64")


def embedding(table, ids, scale: float = 1.0, first: int = 0):
    """``scale * table[ids - first]``, shape ids.shape + [columns], rounded once.

    An id outside ``[first, first + rows)`` gives zeros, so that ranks holding
    slices of a vocabulary (``first``: the slice's first id) add up to the
    whole lookup.
    """
    check_cuda("embedding", table, ids)
    check_type("embedding", "table", table.dtype, REAL)
    _check_ids("embedding", ids)
    if table.dim() != 2:
        raise ValueError("embedding: table must be a matrix")
    table, ids = unit_rows(table), ids.contiguous()
    v, d = table.shape
    out = torch.empty(ids.shape + (d,), dtype=table.dtype, device=table.device)
    ctx, stream = on(table.device)
    with ctx:
        call("ndt_b200_embedding_dev", CODES[table.dtype], table.data_ptr(), v, d, max(d, table.stride(0)), ids.data_ptr(),
             ids.dtype == torch.int64, ids.numel(), first, scale, out.data_ptr(), d, stream)
    return out


def embedding_grad(grad, ids, rows: int, scale: float = 1.0, first: int = 0, out_dtype=None, out=None):
    """The gradient of ``embedding``'s table: ``[rows, columns]`` with row v
    ``scale`` times the sum of grad over the places of id ``first + v``.

    Summed in 32 bits in a fixed order, so equal calls give equal bits.
    ``out_dtype`` defaults to grad's type.  With ``out`` the sums are added to
    it, and only the rows that ids name are touched.
    """
    check_cuda("embedding_grad", grad, ids, out)
    check_type("embedding_grad", "grad", grad.dtype, REAL)
    _check_ids("embedding_grad", ids)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise ValueError("embedding_grad: grad must have the shape of ids and one axis more")
    if rows < 0:
        raise ValueError("embedding_grad: rows must not be negative")
    d = grad.shape[-1]
    g = unit_rows(grad if grad.dim() == 2 else grad.reshape(ids.numel(), d))
    ids = ids.contiguous()
    accumulate = out is not None
    if accumulate:
        check_type("embedding_grad", "out", out.dtype, REAL)
        if out.shape != (rows, d) or (d > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < d):
            raise ValueError("embedding_grad: out must be [rows, columns] with unit stride along the columns")
    else:
        out_dtype = out_dtype or grad.dtype
        check_type("embedding_grad", "out_dtype", out_dtype, REAL)
        out = torch.empty((rows, d), dtype=out_dtype, device=grad.device)
    ctx, stream = on(grad.device)
    with ctx:
        call("ndt_b200_embedding_grad_dev", CODES[g.dtype], g.data_ptr(), max(d, g.stride(0)), ids.data_ptr(),
             ids.dtype == torch.int64, ids.numel(), rows, d, first, scale, CODES[out.dtype], out.data_ptr(),
             max(d, out.stride(0)), accumulate, stream)
    return out


class _Embedding(Function):
    @staticmethod
    def forward(ctx, table, ids, scale, first):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, first, table.dtype)
        return embedding(table, ids, scale, first)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        rows, scale, first, dtype = ctx.args
        return embedding_grad(grad, ids, rows, scale, first, out_dtype=dtype), None, None, None


def torch_embedding(table, ids, scale: float = 1.0, first: int = 0):
    """``embedding`` with autograd (a dense gradient of the table's type)."""
    return _Embedding.apply(table, ids, scale, first)


__all__ = ["embedding", "embedding_grad", "torch_embedding"]
