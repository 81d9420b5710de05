"""The expert layer where values of one token differ by many powers of two.

8-bit weights multiply in float16, and a float16 layer's activations enter the
second product as two float16 parts, each token's row brought into that type's
range by a power of two first.  A channel that dominates its row but meets only
zero weights must not cost the others their bits.
"""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from model_ref import FLOOR, UNIT
from test_gpu_experts import check, gen, layer, normal, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,h,i", [(1, 256, 64), (12, 272, 40), (5, 77, 35)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_channel_that_dominates_the_token(gpu, t, h, i, dtype):
    """x[0] is 2^19 or 2^20 times the rest and its weights are zero, so the
    error bound, which is of |x| |w|, is that of the other channels."""
    router = (normal(gen(1), 4, h) * h ** -0.5).to(dtype)
    w_in, w_out = normal(gen(2), 4, 2 * i, h) * h ** -0.5, normal(gen(3), 4, h, i) * i ** -0.5
    router[:, 0] = 0
    w_in[:, :, 0] = 0
    (w_in, si, vi), (w_out, so, vo) = stored(w_in), stored(w_out)
    x = normal(gen(4), t, h)
    if dtype == torch.float16:
        x *= 2.0 ** -4
    x[:, 0] = 2.0 ** 20 if dtype == torch.bfloat16 else 2.0 ** 15
    check(gpu, x.to(dtype), (router, w_in, w_out, si, so, vi, vo), 2, True)


def test_powers_of_two_are_exact(gpu):
    """x 2^-104 with the router and the scales of w_in 2^104 times larger is the same layer, bit for bit."""
    router, w_in, w_out, si, so, _, _ = layer(6, 144, 40, torch.bfloat16, True, seed=5)
    x = normal(gen(6), 9, 144).to(torch.bfloat16)
    p = 2.0 ** 104
    y, ids, weights = gpu.expert_layer(x, router, w_in, w_out, 2, in_scales=si, out_scales=so)
    z, jds, veights = gpu.expert_layer(x / p, router * p, w_in, w_out, 2, in_scales=si * p, out_scales=so)
    assert torch.equal(ids, jds) and torch.equal(weights, veights) and torch.equal(y, z)


def test_infinity_beside_large_numbers(gpu):
    """An activation beyond float32 and one of 1e15, of opposite weights: the sums are the infinity, as in 32 bits."""
    i, h = 200, 64
    w_in, w_out = torch.zeros(1, 2 * i, h, device="cuda"), torch.zeros(1, h, i, device="cuda")
    w_in[0, [0, 130, i, i + 130], 0] = 1.0  # gate and up of outputs 0 and 130, in three blocks of 128 rows
    w_out[0, :, 0], w_out[0, :, 130] = 1.0, -1.0
    si = torch.tensor([1e30, 1e15, 1.0, 1.0], device="cuda").view(1, 4, 1)
    so = torch.ones(1, 1, 2, device="cuda")
    e4 = torch.float8_e4m3fn
    x = torch.ones(3, h, device="cuda", dtype=torch.bfloat16)
    x[1, 0] = 0.0
    router = torch.zeros(1, h, device="cuda", dtype=torch.bfloat16)
    y, _, _ = gpu.expert_layer(x, router, w_in.to(e4), w_out.to(e4), 1, in_scales=si, out_scales=so)
    assert bool((y[[0, 2]] == float("inf")).all()) and not y[1].any()


@pytest.mark.parametrize("eight", [False, True])
def test_an_activation_that_dominates_its_row(gpu, eight):
    """One of silu(gate) * up is about 2^24 times the rest and meets zero weights."""
    h, i, t, eps = 64, 40, 6, 2.0 ** -23
    dtype = torch.float16
    w_in, w_out = normal(gen(7), 1, 2 * i, h) * h ** -0.5 * 0.5, normal(gen(8), 1, h, i) * i ** -0.5
    w_in[:, [0, i]] = 2.0 ** 7 / h
    w_out[:, :, 0] = 0
    si = so = None
    if eight:
        (w_in, si, vi), (w_out, so, vo) = stored(w_in), stored(w_out)
    else:
        w_in, w_out = w_in.to(dtype), w_out.to(dtype)
        vi, vo = w_in.double(), w_out.double()
    x = (normal(gen(9), t, h).abs() * 8).to(dtype)
    y, _, _ = gpu.expert_layer(x, torch.zeros(1, h, dtype=dtype, device="cuda"), w_in, w_out, 1, in_scales=si, out_scales=so)
    a = x.double() @ vi[0].T
    da = (h + 32) * eps * (x.double().abs() @ vi[0].abs().T)
    g, u, dg, du = a[:, :i], a[:, i:], da[:, :i], da[:, i:]
    s = torch.nn.functional.silu(g)
    b = s * u
    most = b.abs().amax(1, keepdim=True)
    assert bool((most > 2.0 ** 14 * b[:, 1:].abs().median()).all())
    # two parts of 11 bits; the low one ends at 2^-39 of the row's largest
    db = 1.1 * dg * (u.abs() + du) + s.abs() * du + (2.0 ** -21 + 8 * eps) * b.abs() + 2.0 ** -38 * most
    ref = b @ vo[0].T
    bound = db @ vo[0].abs().T + (i + 32) * eps * (b.abs() @ vo[0].abs().T) + UNIT[dtype] * 1.01 * ref.abs() + FLOOR[dtype]
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
