"""The expert layer against a float64 form (model_ref.experts), which also
bounds what the roundings on the way may come to.  A choice has to be the
float64 form's wherever it is clear of the router's rounding, and elsewhere no
chosen expert may lie below an unchosen one by more than that rounding."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from model_ref import experts, quantize, stands_for

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn
HALF = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def stored(w):
    """8-bit weights [e, r, c], their scales, and what they stand for."""
    q, s, v = zip(*((q.float().to(E4), sc.float(), stands_for(q, sc, 128)) for q, sc in (quantize(m, 128, E4) for m in w)))
    return torch.stack(q), torch.stack(s), torch.stack(v)


def layer(e, h, i, dtype, eight, seed=1):
    router = (normal(gen(seed), e, h) * h ** -0.5).to(dtype)
    w_in, w_out = normal(gen(seed + 1), e, 2 * i, h) * h ** -0.5, normal(gen(seed + 2), e, h, i) * i ** -0.5
    if eight:
        (w_in, si, vi), (w_out, so, vo) = stored(w_in), stored(w_out)
        return router, w_in, w_out, si, so, vi, vo
    w_in, w_out = w_in.to(dtype), w_out.to(dtype)
    return router, w_in, w_out, None, None, w_in.double(), w_out.double()


def check(gpu, x, lay, top, renormalize):
    router, w_in, w_out, si, so, vi, vo = lay
    y, ids, weights = gpu.expert_layer(x, router, w_in, w_out, top, in_scales=si, out_scales=so, renormalize=renormalize)
    ry, rids, rw, bound, _, dl = experts(x, router, vi, vo, top, renormalize, ids)
    assert y.dtype == x.dtype and ids.dtype == torch.int32 and weights.dtype == torch.float32
    # (places within the choice may swap where two products are within rounding)
    assert torch.equal(ids.long().sort(1).values, rids.sort(1).values)
    order = torch.gather(rw, 1, rids.argsort(1)), torch.gather(weights.double(), 1, ids.long().argsort(1))
    assert bool(((order[0] - order[1]).abs() <= (4 * dl[:, None] + 2.0 ** -19) * order[0] + 2.0 ** -126).all())
    err = (y.double() - ry).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("weights", ["bf16", "f16", "f8 bf16", "f8 f16"])
@pytest.mark.parametrize("t,e,top,h,i,renormalize", [
    (1, 8, 2, 256, 128, True), (1, 64, 8, 512, 96, True), (1, 1, 1, 64, 64, False), (5, 13, 2, 1000, 200, False),
    (8, 4, 4, 136, 40, True), (9, 3, 1, 72, 264, True), (33, 16, 4, 320, 136, False), (64, 5, 2, 144, 72, True),
    (3, 7, 3, 77, 35, True), (1, 40, 3, 1, 1, False), (40, 2, 1, 131, 130, False)])
def test_layer(gpu, weights, t, e, top, h, i, renormalize):
    dtype = torch.bfloat16 if "bf16" in weights else torch.float16
    lay = layer(e, h, i, dtype, "f8" in weights)
    check(gpu, normal(gen(9), t, h).to(dtype), lay, top, renormalize)


@pytest.mark.parametrize("weights", ["bf16", "f16", "f8 bf16", "f8 f16"])
@pytest.mark.parametrize("t,e,top,h,i,renormalize", [
    (1, 16, 8, 2304, 1056, True), (40, 12, 2, 4352, 320, False), (64, 4, 2, 1088, 2064, True), (3, 12, 4, 2305, 1033, True)])
def test_rows_of_several_stages(gpu, weights, t, e, top, h, i, renormalize):
    """Enough rows for a CTA, and long enough ones, to go round the ring of copies several times."""
    dtype = torch.bfloat16 if "bf16" in weights else torch.float16
    lay = layer(e, h, i, dtype, "f8" in weights, seed=100)
    check(gpu, normal(gen(109), t, h).to(dtype), lay, top, renormalize)


@pytest.mark.parametrize("dtype", HALF)
def test_many_tokens(gpu, dtype):
    """More tokens than one launch's lists take, and more of an expert than a column tile."""
    lay = layer(6, 64, 48, dtype, False, seed=20)
    check(gpu, normal(gen(21), 700, 64).to(dtype), lay, 3, True)


def test_all_tokens_to_one_expert(gpu):
    lay = layer(16, 128, 64, torch.bfloat16, False, seed=30)
    x = normal(gen(31), 50, 128).abs().to(torch.bfloat16)
    router = lay[0].clone()
    router[11] = 1.0
    check(gpu, x, (router,) + lay[1:], 1, True)


def test_many_experts(gpu):
    lay = layer(1024, 32, 8, torch.bfloat16, False, seed=40)
    check(gpu, normal(gen(41), 4, 32).to(torch.bfloat16), lay, 16, True)


def test_ties_go_to_the_lowest_index(gpu):
    router, w_in, w_out, *_ = layer(9, 64, 16, torch.bfloat16, False, seed=50)
    router = torch.zeros_like(router)
    x = normal(gen(51), 3, 64).to(torch.bfloat16)
    _, ids, weights = gpu.expert_layer(x, router, w_in, w_out, 4, renormalize=False)
    assert torch.equal(ids, torch.arange(4, device="cuda", dtype=torch.int32).expand(3, 4))
    assert bool(((weights - 1 / 9).abs() < 1e-7).all())
    router[5] = -0.0
    router[7] = 1.0
    x = x.abs()
    _, ids, _ = gpu.expert_layer(x, router, w_in, w_out, 4)
    assert torch.equal(ids, torch.tensor([7, 0, 1, 2], device="cuda", dtype=torch.int32).expand(3, 4))


@pytest.mark.parametrize("eight", [False, True])
def test_special_values_stay_with_their_tokens(gpu, eight):
    lay = layer(6, 96, 40, torch.bfloat16, eight, seed=60)
    router, w_in, w_out, si, so, vi, vo = lay
    x = normal(gen(61), 12, 96).to(torch.bfloat16)
    y, ids, weights = gpu.expert_layer(x, router, w_in, w_out, 2, in_scales=si, out_scales=so)
    bad = x.clone()
    bad[3, 50], bad[7, 1], bad[8, 2] = float("nan"), float("inf"), -float("inf")
    z, jds, _ = gpu.expert_layer(bad, router, w_in, w_out, 2, in_scales=si, out_scales=so)
    fine = [t for t in range(12) if t not in (3, 7, 8)]
    assert torch.equal(z[fine], y[fine]) and not bool(torch.isfinite(z[[3, 7, 8]]).any())
    assert bool((jds >= 0).all() and (jds < 6).all()) and bool((jds[:, 0] != jds[:, 1]).all())
    # a NaN weight reaches the tokens of its expert only
    w = w_in.float()
    w[int(ids[0, 0]), 5, 7] = float("nan")
    z, _, _ = gpu.expert_layer(x, router, w.to(w_in.dtype), w_out, 2, in_scales=si, out_scales=so)
    hit = (ids == ids[0, 0]).any(1)
    assert bool(torch.isnan(z[hit]).all()) and torch.equal(z[~hit], y[~hit])


def test_float16_activations_out_of_range(gpu):
    """silu(gate) * up beyond 65504 with an output within it."""
    lay = layer(4, 64, 32, torch.float16, False, seed=70)
    router, w_in, w_out, _, _, _, _ = lay
    w_in, w_out = w_in * 400, w_out * 2.0 ** -12
    lay = (router, w_in, w_out, None, None, w_in.double(), w_out.double())
    x = normal(gen(71), 10, 64).to(torch.float16)
    a = torch.einsum("th,erh->ter", x.double(), w_in.double())
    assert float((torch.nn.functional.silu(a[..., :32]) * a[..., 32:]).abs().max()) > 65504
    check(gpu, x, lay, 2, True)


def test_views_shapes_and_streams(gpu):
    lay = layer(5, 64, 24, torch.bfloat16, False, seed=80)
    router, w_in, w_out, *_ = lay
    x = normal(gen(81), 2, 3, 130).to(torch.bfloat16)
    y, ids, weights = gpu.expert_layer(x[..., 1:65], router, w_in, w_out, 2)
    assert y.shape == (2, 3, 64) and ids.shape == weights.shape == (2, 3, 2)
    flat = x[..., 1:65].reshape(6, 64).contiguous()
    check(gpu, flat, lay, 2, True)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        z, _, _ = gpu.expert_layer(flat, router, w_in.transpose(1, 2).contiguous().transpose(1, 2), w_out, 2)
    torch.cuda.synchronize()
    assert torch.equal(z, y.view(6, 64))
    check(gpu, x[..., 0:65][0, :, 1:], lay, 2, True)  # rows that do not start on 16 bytes
    y, ids, weights = gpu.expert_layer(flat[:0], router, w_in, w_out, 2)
    assert y.shape == (0, 64) and ids.shape == weights.shape == (0, 2)


def test_refusals(gpu):
    router, w_in, w_out, *_ = layer(4, 64, 16, torch.bfloat16, False, seed=90)
    x = normal(gen(91), 3, 64).to(torch.bfloat16)
    f = gpu.expert_layer
    for top in (0, 5):
        with pytest.raises(ValueError):
            f(x, router, w_in, w_out, top)
    with pytest.raises(TypeError):
        f(x.float(), router, w_in, w_out, 2)
    with pytest.raises(TypeError):
        f(x, router.float(), w_in, w_out, 2)
    with pytest.raises(TypeError):
        f(x, router, w_in.half(), w_out.half(), 2)
    with pytest.raises(ValueError):
        f(x[:, :32], router, w_in, w_out, 2)
    with pytest.raises(ValueError):
        f(x, router, w_in[:, :31], w_out, 2)
    with pytest.raises(ValueError):
        f(x, router, w_in.to(E4), w_out.to(E4), 2)
    with pytest.raises(ValueError):
        f(x, router, w_in, w_out, 2, in_scales=torch.ones(4, 1, 1, device="cuda"))
    with pytest.raises(ValueError):
        f(x, router, w_in.to(E4), w_out.to(E4), 2, in_scales=torch.ones(4, 2, 1, device="cuda"),
          out_scales=torch.ones(4, 1, 1, device="cuda"))
    with pytest.raises(gpu.NDTensorsError):
        f(x, router.cpu(), w_in, w_out, 2)
    big = torch.zeros(1025, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(gpu.NDTensorsError):
        f(big[:1], big, torch.zeros(1025, 2, 8, dtype=torch.bfloat16, device="cuda"), big.view(1025, 8, 1), 2)
