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
from torch.autograd.function import once_differentiable

from ._model import FLOAT8, REAL, calls, code_of, device_of, launch, no_gradient, out_of, plain, rows_of, written

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
    with ``values=False`` only ``(qt, scales_t)``).  They carry no gradient to
    x: a parameter's 8-bit form is a constant.
    """
    device = device_of("quantize_blocks", x)
    xt, qt8 = code_of("quantize_blocks", "x", x.dtype, REAL), code_of("quantize_blocks", "dtype", dtype, FLOAT8)
    if x.dim() != 2:
        raise ValueError("quantize_blocks: x must be a matrix")
    if block_rows not in (1, 128):
        raise ValueError("quantize_blocks: block_rows must be 1 or 128")
    if not (values or transposed):
        raise ValueError("quantize_blocks: nothing to compute")
    r, c = x.shape
    (x,) = plain(x)
    q = s = t = u = None
    qa = ta = (None, 0, None, 0, 0)
    if values:
        q, s = _empty8(r, c, dtype, x.device), _empty_scales(r, c, block_rows, x.device)
        qa = (q.data_ptr(), max(16, q.stride(0)), s.data_ptr(), s.stride(0), s.stride(1))
    if transposed:
        t, u = _empty8(c, r, dtype, x.device), _empty_scales(c, r, block_rows, x.device)
        ta = (t.data_ptr(), max(16, t.stride(0)), u.data_ptr(), u.stride(0), u.stride(1))
    launch("ndt_b200_quantize_dev", device, xt, x.data_ptr(), r, c, x.stride(0), x.stride(1), block_rows, qt8, *qa, *ta)
    return ((q, s) if values else ()) + ((t, u) if transposed else ())


def _block_rows(what: str, q, s) -> int:
    """Whether the scales are for single rows (1) or for 128 rows."""
    if q.dim() != 2 or s.dim() != 2 or s.dtype != torch.float32:
        raise ValueError(f"{what}: an operand is a float8 matrix with a float32 matrix of scales")
    r, c = q.shape
    rb, kb = s.shape
    if kb == (c + 127) // 128:
        if rb == (r + 127) // 128:
            return 128
        if rb == r:
            return 1
    raise ValueError(f"{what}: scales of shape {tuple(s.shape)} do not fit an operand of shape {tuple(q.shape)}")


def scaled_gemm(a, a_scales, b, b_scales, out_dtype=torch.bfloat16, out=None, accumulate: bool = False):
    """``c[i, j] = sum_k a[i, k] b[j, k]`` of 8-bit a [m, k] and b [n, k].

    Sums are in 32 bits and rounded once to ``out_dtype`` (float32, bfloat16 or
    float16).  ``out`` receives the result, added to what it holds with
    ``accumulate``.  Any strides are taken; rows that do not start on 16 bytes
    cost a copy.  The result carries no gradient, so inputs that require one
    are refused unless gradients are off.
    """
    device = device_of("scaled_gemm", a, a_scales, b, b_scales, out)
    no_gradient("scaled_gemm", "call it under torch.no_grad()", a, a_scales, b, b_scales, out)
    at, bt = code_of("scaled_gemm", "a", a.dtype, FLOAT8), code_of("scaled_gemm", "b", b.dtype, FLOAT8)
    ra, rb = _block_rows("scaled_gemm", a, a_scales), _block_rows("scaled_gemm", b, b_scales)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError("scaled_gemm: the contracted sizes of a and b differ")
    out_of("scaled_gemm", out)
    a, a_scales, b, b_scales = plain(a, a_scales, b, b_scales)
    given = out is not None
    if not given:
        if accumulate:
            raise ValueError("scaled_gemm: accumulate needs out")
        ct = code_of("scaled_gemm", "out_dtype", out_dtype, REAL)
        out = a.new_empty((m, n), dtype=out_dtype)
    else:
        ct = code_of("scaled_gemm", "out", out.dtype, REAL)
        if out.shape != (m, n) or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
            raise ValueError("scaled_gemm: out must be [m, n] with unit stride along n")
    launch("ndt_b200_scaled_gemm_dev", device, m, n, k, at, a.data_ptr(), *a.stride(), ra, a_scales.data_ptr(),
           *a_scales.stride(), bt, b.data_ptr(), *b.stride(), rb, b_scales.data_ptr(), *b_scales.stride(), ct,
           out.data_ptr(), max(n, out.stride(0)), accumulate)
    if given:
        written(out)
    return out


def scaled_linear(x, weight, weight_scales, out_dtype=None):
    """``x w^T`` for activations x [..., k] and stored 8-bit weights w [n, k].

    ``weight_scales`` are those of the 128 x 128 blocks of w.  x is quantised
    in the call (e4m3, a scale for each row and 128 columns).  ``out_dtype``
    defaults to x's type.  The result carries no gradient, so an x that requires
    one is refused unless gradients are off.
    """
    y = calls.scaled_linear(x, weight, weight_scales, out_dtype)
    if y is not None:
        return y
    device = device_of("scaled_linear", x, weight, weight_scales)
    no_gradient("scaled_linear", "use torch_scaled_linear, or call it under torch.no_grad()", x, weight, weight_scales)
    xt = code_of("scaled_linear", "x", x.dtype, REAL)
    wt = code_of("scaled_linear", "weight", weight.dtype, FLOAT8)
    if _block_rows("scaled_linear", weight, weight_scales) != 128:
        raise ValueError("scaled_linear: the weights' scales must be those of 128 x 128 blocks")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError("scaled_linear: the last axis of x does not fit the weights")
    yt = xt if out_dtype is None else code_of("scaled_linear", "out_dtype", out_dtype, REAL)
    x, weight, weight_scales = plain(x, weight, weight_scales)
    x2 = rows_of(x)
    t = x2.shape[0]
    y = x.new_empty(x.shape[:-1] + (n,), dtype=out_dtype or x.dtype)
    launch("ndt_b200_scaled_linear_dev", device, xt, x2.data_ptr(), t, k, *x2.stride(), wt, weight.data_ptr(), n,
           *weight.stride(), weight_scales.data_ptr(), *weight_scales.stride(), yt, y.data_ptr(), n)
    return y


class _ScaledLinear(Function):
    """y = q(x) q(w)^T; dx = q(dy) q(w); dw = q(dy^T) q(x^T)^T, every operand
    quantised along the index that its product contracts."""

    @staticmethod
    def forward(ctx, x, weight, grad_dtype):
        device, xt, wt = x.get_device(), REAL[x.dtype], REAL[weight.dtype]
        n, k = weight.shape
        x2 = rows_of(x)
        t = x2.shape[0]
        y = x.new_empty(x.shape[:-1] + (n,))  # (a view of a matrix could not be changed in place)
        need_x, need_w, _ = ctx.needs_input_grad
        # the weights' 8-bit transpose, kept for x's gradient: values and scales in one buffer
        ld, kb, nb = (n + 15) // 16 * 16, (k + 127) // 128, (n + 127) // 128
        kept = x.new_empty(k * ld + 4 * kb * nb, dtype=torch.uint8) if need_x else None
        at = kept.data_ptr() if need_x else 0
        launch("ndt_b200_scaled_linear_fwd_dev", device, xt, x2.data_ptr(), t, k, *x2.stride(), wt, weight.data_ptr(), n,
               *weight.stride(), y.data_ptr(), max(1, n), at or None, ld, at + k * ld if need_x else None)
        ctx.save_for_backward(x2 if need_w else None, kept)
        ctx.args = device, xt, FLOAT8[grad_dtype], x.shape, weight.shape, weight.dtype, x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        # (once_differentiable costs as much as the call; only a graph of the gradient needs it)
        return _once(ctx, dy) if torch.is_grad_enabled() else _ScaledLinear.grads(ctx, dy)

    @staticmethod
    def grads(ctx, dy):
        x2, kept = ctx.saved_tensors
        device, xt, g8, x_shape, (n, k), w_dtype, x_dtype = ctx.args
        need_x, need_w, _ = ctx.needs_input_grad
        dy2 = rows_of(dy.resolve_neg())
        t = dy2.shape[0]
        ld = (n + 15) // 16 * 16
        dx = dy.new_empty((t, k), dtype=x_dtype) if need_x else None
        dw = dy.new_empty((n, k), dtype=w_dtype) if need_w else None
        launch("ndt_b200_scaled_linear_vjp_dev", device, xt, dy2.data_ptr(), t, n, *dy2.stride(),
               x2.data_ptr() if need_w else None, k, *(x2.stride() if need_w else (0, 0)),
               kept.data_ptr() if need_x else None, ld, kept.data_ptr() + k * ld if need_x else None, g8,
               dx.data_ptr() if need_x else None, max(1, k), REAL[w_dtype], dw.data_ptr() if need_w else None, max(1, k))
        return dx if dx is None or len(x_shape) == 2 else dx.view(x_shape), dw, None


_once = once_differentiable(_ScaledLinear.grads)


def torch_scaled_linear(x, weight, grad_dtype=E4M3):
    """``x w^T`` with autograd, all three products of a training step in 8 bits.

    x [..., k] and weight [n, k] are float32, bfloat16 or float16.  In the
    output and in x's gradient w has a scale for each 128 x 128 block; every
    other operand has one for each 128 elements along the contracted index.
    ``grad_dtype`` is the 8-bit type of the output's gradient (e4m3 or e5m2).
    The result has x's type, the gradients their tensors' types.
    """
    y = calls.torch_scaled_linear(x, weight, grad_dtype)
    if y is not None:
        return y
    device_of("torch_scaled_linear", x, weight)
    code_of("torch_scaled_linear", "x", x.dtype, REAL)
    code_of("torch_scaled_linear", "weight", weight.dtype, REAL)
    code_of("torch_scaled_linear", "grad_dtype", grad_dtype, FLOAT8)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("torch_scaled_linear: the last axis of x does not fit the weights")
    return _ScaledLinear.apply(*plain(x, weight), grad_dtype)


__all__ = ["quantize_blocks", "scaled_gemm", "scaled_linear", "torch_scaled_linear"]
