"""Plain float64 forms of the language-model operators, for the tests."""

from __future__ import annotations

import torch

TINY = 2.0 ** -100
FMAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
#: half the distance between neighbouring numbers, relative
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
#: below this a float16 has fewer bits: half its smallest step
FLOOR = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def round8(v, dtype):
    """float64 to the nearest value of an 8-bit type (ties to even, saturated; NaN and infinities as the type has them)."""
    mantissa, low = (3, -6) if dtype == torch.float8_e4m3fn else (2, -14)
    m, e = torch.frexp(torch.where(torch.isfinite(v), v, torch.ones_like(v)).abs().clamp(min=2.0 ** -40))
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=low) - mantissa)
    r = (torch.round(v / step) * step).clamp(-FMAX[dtype], FMAX[dtype])
    inf = torch.isinf(v)
    if dtype == torch.float8_e4m3fn:
        return torch.where(inf | torch.isnan(v), torch.full_like(v, float("nan")), r)
    return torch.where(inf | torch.isnan(v), v, r)


def quantize(x, block_rows, dtype):
    """(values, scales) of x [r, c] in float64."""
    r, c = x.shape
    x = x.double()
    rb, cb = -(-r // block_rows), -(-c // 128)
    p = torch.zeros(rb * block_rows, cb * 128, dtype=torch.float64, device=x.device)
    p[:r, :c] = x
    p = p.view(rb, block_rows, cb, 128)
    mag = torch.where(torch.isfinite(p), p.abs(), torch.zeros_like(p))
    s = (mag.amax((1, 3)).clamp(min=TINY) / FMAX[dtype]).float().double()
    quotient = (p / s[:, None, :, None]).float().double()
    q = round8(torch.where(torch.isfinite(p), quotient, p), dtype)
    return q.reshape(rb * block_rows, cb * 128)[:r, :c], s


def stands_for(q, s, block_rows):
    """float64 values of an 8-bit matrix with scales."""
    r, c = q.shape
    full = s.double().repeat_interleave(128, 1)[:, :c]
    full = full.repeat_interleave(block_rows, 0)[:r] if block_rows > 1 else full
    return q.float().double() * full


def product_bound(a, b, c, out_dtype):
    """How far a 32-bit sum of k products, truncated at every step, and its rounding may be from c = a b^T."""
    k = a.shape[1]
    return (k + k // 128 + 8) * 2.0 ** -23 * (a.abs() @ b.abs().T) + UNIT[out_dtype] * c.abs() * 1.01 + FLOOR[out_dtype]


def experts(x, router, w_in, w_out, top, renormalize, chosen=None):
    """y, ids, weights, a bound on y's error, whether each token's choice is clear of the router's rounding, and
    that rounding, from float64 weights.  ``chosen`` [tokens, top]: the experts to sum over (sorted by place) where
    the choice is not clear."""
    dtype = x.dtype
    x, router = x.double(), router.double()
    h, i = router.shape[1], w_out.shape[2]
    logits = x @ router.T
    dl = (h + 8) * 2.0 ** -23 * (x.abs() @ router.abs().T).amax(1)
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    ids = order.indices[:, :top]
    if top == router.shape[0]:
        clear = torch.ones(x.shape[0], dtype=torch.bool, device=x.device)
    else:
        clear = order.values[:, top - 1] - order.values[:, top] > 2 * dl
    if chosen is not None:
        least = torch.gather(logits, 1, chosen.long()).amin(1)
        assert bool((least >= order.values[:, top - 1] - 2 * dl).all()), "an expert was chosen before a larger one"
        ids = torch.where(clear[:, None], ids, chosen.long())
    p = torch.softmax(logits, 1)
    weights = torch.gather(p, 1, ids)
    if renormalize:
        weights = weights / weights.sum(1, keepdim=True)
    y = torch.zeros_like(x)
    err = torch.zeros_like(x)
    eps = 2.0 ** -23
    split = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -20
    for e in range(router.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not len(t):
            continue
        a = x[t] @ w_in[e].T
        da = (h + 32) * eps * (x[t].abs() @ w_in[e].abs().T)
        g, u, dg, du = a[:, :i], a[:, i:], da[:, :i], da[:, i:]
        s = torch.nn.functional.silu(g)
        b = s * u
        db = 1.1 * dg * (u.abs() + du) + s.abs() * du + (split + 8 * eps) * b.abs()
        if dtype == torch.float16:  # the scaled low part ends at 2^-24 of the largest
            db = db + 2.0 ** -23 * b.abs().amax(1, keepdim=True)
        w = weights[t, j][:, None]
        o, size = b @ w_out[e].T, b.abs() @ w_out[e].abs().T
        y.index_add_(0, t, w * o)
        dw = 2 * dl[t][:, None] * 2 + 16 * eps
        err.index_add_(0, t, w * (db @ w_out[e].abs().T + ((i + 32) * eps + dw) * size))
    err = err + UNIT[dtype] * 1.01 * y.abs() + FLOOR[dtype]
    return y, ids, weights, err, clear, dl
