"""Products of 8-bit floating-point matrices with a scale for each block of 128.

An 8-bit matrix is a pair: float8 values ``q [rows, columns]`` and float32
``scales`` of its blocks, ``[rows, ceil(columns / 128)]`` for blocks of 1 x 128
or ``[ceil(rows / 128), ceil(columns / 128)]`` for blocks of 128 x 128.  It
stands for ``q * scale``.  Everything runs on torch's current stream.

``quantize_blocks`` makes such pairs, ``scaled_gemm`` multiplies two of them,
``scaled_linear`` is a layer with stored 8-bit weights, ``torch_scaled_linear``
a trained layer whose product and gradients all run in 8 bits.
"""

from __future__ import annotations

import torch
from torch.autograd import Function

from ._model import CODES, FLOAT8, REAL, call, check_cuda, check_type, on, rows_of
from .tensor import NDTensorsError

E4M3 = torch.float8_e4m3fn


def _empty8(rows: int, cols: int, dtype, device):
    """An uninitialised 8-bit matrix whose rows start on 16 bytes."""
    ld = (cols + 15) // 16 * 16
    q = torch.empty((rows, ld), dtype=dtype, device=device)
    return q if ld == cols else q[:, :cols]


def _empty_scales(rows: int, cols: int, block_rows: int, device):
    """Uninitialised scales of a [rows, cols] matrix, stored column by column (the order the product reads them in)."""
    rb = rows if block_rows == 1 else (rows + 127) // 128
    return torch.empty(((cols + 127) // 128, rb), dtype=torch.float32, device=device).t()


def quantize_blocks(x, block_rows: int = 1, dtype=E4M3, transposed: bool = False, values: bool = True):
    """The 8-bit form of a matrix x (float32, bfloat16 or float16).

    Blocks are ``block_rows`` (1 or 128) x 128.  The scale of a block is its
    largest finite magnitude (at least 2^-100) over the type's largest value;
    an element is its quotient with the scale, rounded to nearest.  NaN stays
    NaN, an infinity becomes e5m2's or, in e4m3, NaN.

    Returns ``(q, scales)``; with ``transposed`` ``(q, scales, qt, scales_t)``,
    qt being the 8-bit form of x's transpose from the same pass over x (and
    with ``values=False`` only ``(qt, scales_t)``).
    """
    check_cuda("quantize_blocks", x)
    check_type("quantize_blocks", "x", x.dtype, REAL)
    check_type("quantize_blocks", "dtype", dtype, FLOAT8)
    if x.dim() != 2:
        raise ValueError("quantize_blocks: x must be a matrix")
    if block_rows not in (1, 128):
        raise ValueError("quantize_blocks: block_rows must be 1 or 128")
    if not (values or transposed):
        raise ValueError("quantize_blocks: nothing to compute")
    r, c = x.shape
    q = s = t = u = None
    qa = ta = (None, 0, None, 0, 0)
    if values:
        q, s = _empty8(r, c, dtype, x.device), _empty_scales(r, c, block_rows, x.device)
        qa = (q.data_ptr(), max(16, q.stride(0)), s.data_ptr(), s.stride(0), s.stride(1))
    if transposed:
        t, u = _empty8(c, r, dtype, x.device), _empty_scales(c, r, block_rows, x.device)
        ta = (t.data_ptr(), max(16, t.stride(0)), u.data_ptr(), u.stride(0), u.stride(1))
    ctx, stream = on(x.device)
    with ctx:
        call("ndt_b200_quantize_dev", CODES[x.dtype], x.data_ptr(), r, c, x.stride(0), x.stride(1), block_rows, CODES[dtype],
             *qa, *ta, stream)
    return ((q, s) if values else ()) + ((t, u) if transposed else ())


def _block_rows(what: str, q, s):
    """Whether the scales are for single rows (1) or for 128 rows."""
    check_type(what, "an 8-bit operand", q.dtype, FLOAT8)
    if q.dim() != 2 or s.dim() != 2 or s.dtype != torch.float32:
        raise ValueError(f"{what}: an operand is a float8 matrix with a float32 matrix of scales")
    r, kb = q.shape[0], (q.shape[1] + 127) // 128
    if s.shape[1] == kb:
        if s.shape[0] == (r + 127) // 128:
            return 128
        if s.shape[0] == r:
            return 1
    raise ValueError(f"{what}: scales of shape {tuple(s.shape)} do not fit an operand of shape {tuple(q.shape)}")


def scaled_gemm(a, a_scales, b, b_scales, out_dtype=torch.bfloat16, out=None, accumulate: bool = False):
    """``c[i, j] = sum_k a[i, k] b[j, k]`` of 8-bit a [m, k] and b [n, k].

    Sums are in 32 bits and rounded once to ``out_dtype`` (float32, bfloat16 or
    float16).  ``out`` receives the result, added to what it holds with
    ``accumulate``.  Any strides are taken; rows that do not start on 16 bytes
    cost a copy.
    """
    check_cuda("scaled_gemm", a, a_scales, b, b_scales, out)
    ra, rb = _block_rows("scaled_gemm", a, a_scales), _block_rows("scaled_gemm", b, b_scales)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError("scaled_gemm: the contracted sizes of a and b differ")
    if out is None:
        if accumulate:
            raise ValueError("scaled_gemm: accumulate needs out")
        check_type("scaled_gemm", "out_dtype", out_dtype, REAL)
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    else:
        check_type("scaled_gemm", "out", out.dtype, REAL)
        if out.shape != (m, n) or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
            raise ValueError("scaled_gemm: out must be [m, n] with unit stride along n")
    ctx, stream = on(a.device)
    with ctx:
        call("ndt_b200_scaled_gemm_dev", m, n, k, CODES[a.dtype], a.data_ptr(), a.stride(0), a.stride(1), ra,
             a_scales.data_ptr(), a_scales.stride(0), a_scales.stride(1), CODES[b.dtype], b.data_ptr(), b.stride(0),
             b.stride(1), rb, b_scales.data_ptr(), b_scales.stride(0), b_scales.stride(1), CODES[out.dtype],
             out.data_ptr(), max(n, out.stride(0)), int(accumulate), stream)
    return out


def scaled_linear(x, weight, weight_scales, out_dtype=None):
    """``x w^T`` for activations x [..., k] and stored 8-bit weights w [n, k].

    ``weight_scales`` are those of the 128 x 128 blocks of w.  x is quantised
    in the call (e4m3, a scale for each row and 128 columns).  ``out_dtype``
    defaults to x's type.
    """
    check_cuda("scaled_linear", x, weight, weight_scales)
    check_type("scaled_linear", "x", x.dtype, REAL)
    if _block_rows("scaled_linear", weight, weight_scales) != 128:
        raise ValueError("scaled_linear: the weights' scales must be those of 128 x 128 blocks")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError("scaled_linear: the last axis of x does not fit the weights")
    out_dtype = out_dtype or x.dtype
    check_type("scaled_linear", "out_dtype", out_dtype, REAL)
    x2 = rows_of(x)
    t = x2.shape[0]
    y = torch.empty((t, n), dtype=out_dtype, device=x.device)
    ctx, stream = on(x.device)
    with ctx:
        call("ndt_b200_scaled_linear_dev", CODES[x.dtype], x2.data_ptr(), t, k, x2.stride(0), x2.stride(1),
             CODES[weight.dtype], weight.data_ptr(), n, weight.stride(0), weight.stride(1), weight_scales.data_ptr(),
             weight_scales.stride(0), weight_scales.stride(1), CODES[out_dtype], y.data_ptr(), n, stream)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (n,))


class _ScaledLinear(Function):
    """y = q(x) q(w)^T; dx = q(dy) q(w); dw = q(dy^T) q(x^T)^T, every operand
    quantised along the index that its product contracts."""

    @staticmethod
    def forward(ctx, x, weight, grad_dtype):
        x2 = rows_of(x)
        xq, xs = quantize_blocks(x2)
        ctx.needs = ctx.needs_input_grad
        if ctx.needs[0]:
            wq, ws, wt, wu = quantize_blocks(weight, 128, transposed=True)
        else:
            (wq, ws), wt, wu = quantize_blocks(weight, 128), None, None
        ctx.save_for_backward(x2 if ctx.needs[1] else None, wt, wu)
        ctx.grad_dtype, ctx.x_shape, ctx.types = grad_dtype, x.shape, (x.dtype, weight.dtype)
        y = scaled_gemm(xq, xs, wq, ws, out_dtype=x.dtype)
        return y if x.dim() == 2 else y.view(x.shape[:-1] + (weight.shape[0],))

    @staticmethod
    def backward(ctx, dy):
        x2, wt, wu = ctx.saved_tensors
        dx = dw = None
        dy2 = rows_of(dy)
        if ctx.needs[0] and ctx.needs[1]:
            gq, gs, gt, gu = quantize_blocks(dy2, 1, ctx.grad_dtype, transposed=True)
        elif ctx.needs[0]:
            gq, gs = quantize_blocks(dy2, 1, ctx.grad_dtype)
        elif ctx.needs[1]:
            gt, gu = quantize_blocks(dy2, 1, ctx.grad_dtype, transposed=True, values=False)
        if ctx.needs[0]:
            dx = scaled_gemm(gq, gs, wt, wu, out_dtype=ctx.types[0])
            dx = dx if len(ctx.x_shape) == 2 else dx.view(ctx.x_shape)
        if ctx.needs[1]:
            xt, xu = quantize_blocks(x2, transposed=True, values=False)
            dw = scaled_gemm(gt, gu, xt, xu, out_dtype=ctx.types[1])
        return dx, dw, None


def torch_scaled_linear(x, weight, grad_dtype=E4M3):
    """``x w^T`` with autograd, all three products of a training step in 8 bits.

    x [..., k] and weight [n, k] are float32, bfloat16 or float16.  In the
    output and in x's gradient w has a scale for each 128 x 128 block; every
    other operand has one for each 128 elements along the contracted index.
    ``grad_dtype`` is the 8-bit type of the output's gradient (e4m3 or e5m2).
    The result has x's type, the gradients their tensors' types.
    """
    check_cuda("torch_scaled_linear", x, weight)
    check_type("torch_scaled_linear", "x", x.dtype, REAL)
    check_type("torch_scaled_linear", "weight", weight.dtype, REAL)
    check_type("torch_scaled_linear", "grad_dtype", grad_dtype, FLOAT8)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("torch_scaled_linear: the last axis of x does not fit the weights")
    return _ScaledLinear.apply(x, weight, grad_dtype)


__all__ = ["quantize_blocks", "scaled_gemm", "scaled_linear", "torch_scaled_linear", "NDTensorsError"]
