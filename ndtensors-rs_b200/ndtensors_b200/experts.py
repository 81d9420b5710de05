"""A mixture-of-experts layer for a few tokens: a block-sparse contraction
whose blocks the data choose, in one kernel on torch's current stream."""

from __future__ import annotations

import torch

from ._model import code_of, device_of, launch, no_gradient, plain, rows_of, unit_rows

E4M3 = torch.float8_e4m3fn
_HALF = {torch.bfloat16: 3, torch.float16: 4}
_F32 = {torch.float32: 2}


def expert_layer(x, router, w_in, w_out, top: int, in_scales=None, out_scales=None, renormalize: bool = True):
    """The layer's output for x [..., h], and each token's choice.

    ``router`` is [experts, h], ``w_in`` [experts, 2 i, h] (gate rows, then up
    rows), ``w_out`` [experts, h, i].  A token goes to the ``top`` experts of
    its largest router products (ties to the lowest index), weighted by their
    softmax over all experts, divided by the sum of the chosen with
    ``renormalize``; an expert computes ``w_out (silu(gate) * up)``.

    x is bfloat16 or float16, router too; the experts' weights have x's type or
    are float8 e4m3 with the float32 scales of their 128 x 128 blocks
    (``in_scales`` [experts, ceil(2 i / 128), ceil(h / 128)], ``out_scales``
    [experts, ceil(h / 128), ceil(i / 128)]).

    Returns ``(y, ids, weights)``: x's shape and type, and int32 / float32
    [..., top].  They carry no gradient, so inputs that require one are refused
    unless gradients are off.  Made for at most about a hundred tokens (a decoding batch);
    more are right, but an expert's weights are read anew for each group of its
    tokens: 8 (or 16) where their rows are short, and as many as fit 119 KB of
    shared memory at max(2 h, 4 i) bytes each where they are long (8 up to h 7424
    and i 3712, 4 for i 6400, 2 for i 14336; fewer for 8-bit weights or odd lengths).
    """
    device = device_of("expert_layer", x, router, w_in, w_out, in_scales, out_scales)
    no_gradient("expert_layer", "call it under torch.no_grad()", x, router, w_in, w_out, in_scales, out_scales)
    xt = code_of("expert_layer", "x", x.dtype, _HALF)
    code_of("expert_layer", "router", router.dtype, {x.dtype: xt})
    wt = code_of("expert_layer", "w_in", w_in.dtype, {x.dtype: xt, E4M3: 5})
    code_of("expert_layer", "w_out", w_out.dtype, {w_in.dtype: wt})
    if router.dim() != 2 or w_in.dim() != 3 or w_out.dim() != 3 or x.dim() < 1:
        raise ValueError("expert_layer: router is a matrix, w_in and w_out have three axes")
    e, h = router.shape
    i = w_out.shape[2]
    if x.shape[-1] != h or w_in.shape != (e, 2 * i, h) or w_out.shape != (e, h, i):
        raise ValueError("expert_layer: the sizes of x, router, w_in and w_out do not fit")
    if not 1 <= top <= e:
        raise ValueError("expert_layer: top must be from 1 to the number of experts")
    x, router, w_in, w_out, in_scales, out_scales = plain(x, router, w_in, w_out, in_scales, out_scales)
    if w_in.dtype == E4M3:
        if in_scales is None or out_scales is None:
            raise ValueError("expert_layer: float8 weights need in_scales and out_scales")
        hb, ib, jb = (h + 127) // 128, (i + 127) // 128, (2 * i + 127) // 128
        if in_scales.shape != (e, jb, hb) or out_scales.shape != (e, hb, ib):
            raise ValueError("expert_layer: scales do not fit the weights' 128 x 128 blocks")
        code_of("expert_layer", "in_scales", in_scales.dtype, _F32)
        code_of("expert_layer", "out_scales", out_scales.dtype, _F32)
        in_scales, out_scales = in_scales.contiguous(), out_scales.contiguous()
    elif in_scales is not None or out_scales is not None:
        raise ValueError("expert_layer: scales are for float8 weights")
    x2 = unit_rows(rows_of(x))
    router, w_in, w_out = router.contiguous(), w_in.contiguous(), w_out.contiguous()
    t = x2.shape[0]
    y = x.new_empty((t, h))
    ids, weights = x.new_empty((t, top), dtype=torch.int32), x.new_empty((t, top), dtype=torch.float32)
    launch("ndt_b200_expert_layer_dev", device, xt, x2.data_ptr(), t, h, max(h, x2.stride(0)), router.data_ptr(), e, wt,
           w_in.data_ptr(), None if in_scales is None else in_scales.data_ptr(), w_out.data_ptr(),
           None if out_scales is None else out_scales.data_ptr(), i, top, renormalize, y.data_ptr(), h, ids.data_ptr(),
           weights.data_ptr())
    lead = x.shape[:-1]
    return (y, ids, weights) if x.dim() == 2 else (y.view(x.shape), ids.view(lead + (top,)), weights.view(lead + (top,)))


__all__ = ["expert_layer"]
