"""Embedding lookup with scaling, and its gradient: contraction with a one-hot
tensor that is never formed.  Everything runs on torch's current stream."""

from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._model import REAL, calls, code_of, device_of, launch, no_gradient, out_of, plain, unit_rows, written

_IDS = {torch.int32: 0, torch.int64: 1}


def embedding(table, ids, scale: float = 1.0, first: int = 0):
    """``scale * table[ids - first]``, shape ids.shape + [columns], rounded once.

    An id outside ``[first, first + rows)`` gives zeros, so that ranks holding
    slices of a vocabulary (``first``: the slice's first id) add up to the
    whole lookup.  The result carries no gradient (``torch_embedding`` has one),
    so a table that requires one is refused unless gradients are off.
    """
    out = calls.embedding(table, ids, scale, first)
    if out is not None:
        return out
    device_of("embedding", table, ids)
    no_gradient("embedding", "use torch_embedding, or call it under torch.no_grad()", table)
    return _lookup(table, ids, scale, first)


def _lookup(table, ids, scale, first):
    device = device_of("embedding", table, ids)
    tt, it = code_of("embedding", "table", table.dtype, REAL), code_of("embedding", "ids", ids.dtype, _IDS)
    if table.dim() != 2:
        raise ValueError("embedding: table must be a matrix")
    table, ids = plain(table, ids)
    table, ids = unit_rows(table), ids.contiguous()
    v, d = table.shape
    out = table.new_empty(ids.shape + (d,))
    launch("ndt_b200_embedding_dev", device, tt, table.data_ptr(), v, d, max(d, table.stride(0)), ids.data_ptr(), it,
           ids.numel(), first, scale, out.data_ptr(), d)
    return out


def embedding_grad(grad, ids, rows: int, scale: float = 1.0, first: int = 0, out_dtype=None, out=None):
    """The gradient of ``embedding``'s table: ``[rows, columns]`` with row v
    ``scale`` times the sum of grad over the places of id ``first + v``.

    Summed in 32 bits in a fixed order, so equal calls give equal bits.
    ``out_dtype`` defaults to grad's type.  With ``out`` the sums are added to
    it, and only the rows that ids name are touched.
    """
    device = device_of("embedding_grad", grad, ids, out)
    no_gradient("embedding_grad", "call it under torch.no_grad()", grad, out)
    gt, it = code_of("embedding_grad", "grad", grad.dtype, REAL), code_of("embedding_grad", "ids", ids.dtype, _IDS)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise ValueError("embedding_grad: grad must have the shape of ids and one axis more")
    if rows < 0:
        raise ValueError("embedding_grad: rows must not be negative")
    out_of("embedding_grad", out)
    grad, ids = plain(grad, ids)
    d, n = grad.shape[-1], ids.numel()
    g = unit_rows(grad if grad.dim() == 2 else grad.reshape(n, d))
    ids = ids.contiguous()
    accumulate = out is not None
    if accumulate:
        ot = code_of("embedding_grad", "out", out.dtype, REAL)
        if out.shape != (rows, d) or (d > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < d):
            raise ValueError("embedding_grad: out must be [rows, columns] with unit stride along the columns")
    else:
        out_dtype = out_dtype or grad.dtype
        ot = code_of("embedding_grad", "out_dtype", out_dtype, REAL)
        out = grad.new_empty((rows, d), dtype=out_dtype)
    launch("ndt_b200_embedding_grad_dev", device, gt, g.data_ptr(), max(d, g.stride(0)), ids.data_ptr(), it, n, rows, d,
           first, scale, ot, out.data_ptr(), max(d, out.stride(0)), accumulate)
    if accumulate:
        written(out)
    return out


class _Embedding(Function):
    @staticmethod
    def forward(ctx, table, ids, scale, first):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, first, table.dtype)
        return _lookup(table, ids, scale, first)

    @staticmethod
    def backward(ctx, grad):
        # (once_differentiable costs as much as the call; only a graph of the gradient needs it)
        return _once(ctx, grad) if torch.is_grad_enabled() else _Embedding.grads(ctx, grad)

    @staticmethod
    def grads(ctx, grad):
        (ids,) = ctx.saved_tensors
        rows, scale, first, dtype = ctx.args
        return embedding_grad(grad, ids, rows, scale, first, out_dtype=dtype), None, None, None


_once = once_differentiable(_Embedding.grads)


def torch_embedding(table, ids, scale: float = 1.0, first: int = 0):
    """``embedding`` with autograd (a dense gradient of the table's type)."""
    out = calls.torch_embedding(table, ids, scale, first)
    return _Embedding.apply(*plain(table, ids), scale, first) if out is None else out


__all__ = ["embedding", "embedding_grad", "torch_embedding"]
