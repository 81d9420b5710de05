"""Embedding lookup and its gradient against float64 forms.

A looked-up value is one product, rounded once.  A gradient row may differ by
the rounding of its 32-bit sum (one 2^-24 of the terms' magnitudes for each
addition) and of its result.
"""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from model_ref import FLOOR, UNIT

pytestmark = pytest.mark.gpu

REAL = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def lookup(table, ids, scale, first):
    row = ids.long() - first
    on = (row >= 0) & (row < table.shape[0])
    out = table.double()[row.clamp(0, max(0, table.shape[0] - 1))] * scale if table.shape[0] else torch.zeros(
        ids.shape + table.shape[1:], dtype=torch.float64, device="cuda")
    return torch.where(on[..., None], out, torch.zeros_like(out))


def scatter(grad, ids, rows, scale, first):
    """(sum, sum of magnitudes, largest count) in float64."""
    row = ids.reshape(-1).long() - first
    on = (row >= 0) & (row < rows)
    g = grad.reshape(-1, grad.shape[-1]).double()[on]
    out = torch.zeros(rows, grad.shape[-1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    out.index_put_((row[on],), g, accumulate=True)
    mag.index_put_((row[on],), g.abs(), accumulate=True)
    count = torch.zeros(rows, dtype=torch.float64, device="cuda").index_put_((row[on],), torch.ones_like(row[on], dtype=torch.float64), accumulate=True)
    return out * scale, mag * abs(scale), count


def check_grad(got, grad, ids, scale=1.0, first=0, base=None):
    ref, mag, count = scatter(grad, ids, got.shape[0], scale, first)
    add = 0.0
    if base is not None:
        ref = ref + base.double()
        add = 2.0 ** -23 * base.double().abs()
    bound = (count[:, None] + 4) * 2.0 ** -24 * mag + add + UNIT[got.dtype] * 1.01 * ref.abs() + FLOOR[got.dtype]
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("dtype", REAL)
@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("v,d,shape", [(1, 1, (1,)), (100, 64, (7,)), (1000, 771, (3, 5)), (50, 2048, (16,)), (33, 24, (400,)),
                                       (10, 1032, (2000,)), (10, 8, (0,))])
def test_lookup(gpu, dtype, ids_type, v, d, shape):
    table = normal(gen(1), v, d).to(dtype)
    ids = torch.randint(0, v, shape, generator=gen(2), device="cuda").to(ids_type)
    out = gpu.embedding(table, ids, scale=27.75)
    ref = lookup(table, ids, 27.75, 0)
    assert out.shape == shape + (d,) and out.dtype == dtype
    assert bool(((out.double() - ref).abs() <= UNIT[dtype] * (1 + 2.0 ** -10) * ref.abs() + FLOOR[dtype]).all())
    assert torch.equal(gpu.embedding(table, ids), table[ids.long()])


def test_lookup_slices_of_a_vocabulary_add_up(gpu):
    table = normal(gen(3), 90, 40)
    ids = torch.randint(0, 90, (300,), generator=gen(4), device="cuda")
    parts = [gpu.embedding(table[lo : lo + 30], ids, first=lo) for lo in (0, 30, 60)]
    assert torch.equal(parts[0] + parts[1] + parts[2], table[ids])
    extreme = torch.tensor([-1, 90, -(2 ** 63), 2 ** 63 - 1, 2 ** 40, 89], device="cuda")
    out = gpu.embedding(table, extreme, first=0)
    assert not out[:5].any() and torch.equal(out[5], table[89])


def test_lookup_views_and_special_values(gpu):
    wide = normal(gen(5), 40, 100).to(torch.bfloat16)
    ids = torch.randint(0, 40, (4, 6), generator=gen(6), device="cuda")
    assert torch.equal(gpu.embedding(wide[:, 3:90], ids.T), wide[:, 3:90][ids.T])
    assert torch.equal(gpu.embedding(wide[:, ::2], ids), wide[:, ::2][ids])
    assert torch.equal(gpu.embedding(wide[1:], ids, first=1)[ids > 0], wide[ids[ids > 0]])
    wide[7, 5], wide[8, 6] = float("nan"), float("inf")
    out = gpu.embedding(wide, torch.tensor([7, 8, 9, 40], device="cuda"), scale=0.5)
    assert bool(torch.isnan(out[0, 5])) and bool(torch.isinf(out[1, 6])) and int((~torch.isfinite(out)).sum()) == 2


def test_lookup_past_32_bit_offsets(gpu):
    """A table of more than 2^31 elements."""
    v, d = 1050000, 2056
    table = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    table[-1] = 3.0
    table[v - 2, 5] = 2.0
    ids = torch.tensor([v - 1, 0, v - 2], device="cuda")
    out = gpu.embedding(table, ids)
    assert bool((out[0] == 3).all()) and not out[1].any() and float(out[2, 5]) == 2 and float(out[2].sum()) == 2
    del table
    g = gpu.embedding_grad(torch.ones(3, d, dtype=torch.bfloat16, device="cuda"), ids, v)
    assert bool((g[-1] == 1).all()) and bool((g[v - 2] == 1).all()) and float(g[1:-2].abs().amax()) == 0


IDS = {
    "spread": lambda n, v: torch.randint(0, v, (n,), generator=gen(7), device="cuda"),
    "one id": lambda n, v: torch.full((n,), v - 1, device="cuda"),
    "few ids": lambda n, v: torch.randint(0, min(v, 3), (n,), generator=gen(8), device="cuda") * ((v - 1) // 3),
    "sorted": lambda n, v: torch.randint(0, v, (n,), generator=gen(9), device="cuda").sort().values,
    "half outside": lambda n, v: torch.randint(-v, v, (n,), generator=gen(10), device="cuda"),
    "all outside": lambda n, v: torch.full((n,), v, device="cuda"),
}


@pytest.mark.parametrize("kind", list(IDS))
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (31, 5, 8), (32, 5, 8), (33, 700, 771), (1000, 40, 64), (3001, 5003, 100),
                                   (20000, 300, 24), (9000, 200000, 8), (0, 50, 16)])
def test_gradient(gpu, kind, n, v, d):
    ids = IDS[kind](n, v)
    grad = normal(gen(11), n, d)
    check_grad(gpu.embedding_grad(grad, ids, v, scale=1.5), grad, ids, 1.5)


@pytest.mark.parametrize("gtype", REAL)
@pytest.mark.parametrize("otype", REAL)
@pytest.mark.parametrize("d", [64, 77])
def test_gradient_types(gpu, gtype, otype, d):
    n, v = 700, 60
    ids = IDS["few ids"](n, v).to(torch.int32)
    grad = normal(gen(12), n, d).to(gtype)
    check_grad(gpu.embedding_grad(grad, ids, v, out_dtype=otype, scale=0.25), grad, ids, 0.25)
    base = normal(gen(13), v, d).to(otype)
    out = base.clone()
    assert gpu.embedding_grad(grad, ids, v, scale=0.25, out=out) is out
    check_grad(out, grad, ids, 0.25, base=base)


def test_gradient_views(gpu):
    n, v, d = 500, 90, 48
    ids = IDS["spread"](2 * n, v)[::2]
    grad = normal(gen(14), n, 2 * d)
    check_grad(gpu.embedding_grad(grad[:, ::2], ids, v), grad[:, ::2], ids)
    check_grad(gpu.embedding_grad(grad[:, 5 : 5 + d], ids, v), grad[:, 5 : 5 + d], ids)
    check_grad(gpu.embedding_grad(grad[:1, :d].expand(n, d), ids, v), grad[:1, :d].expand(n, d), ids)
    check_grad(gpu.embedding_grad(grad[:, :d].contiguous().view(20, 25, d), ids.view(20, 25), v), grad[:, :d], ids)
    wide = torch.full((v, d + 6), 5.0, device="cuda")
    gpu.embedding_grad(grad[:, :d], ids, v, out=wide[:, 3 : 3 + d], first=2)
    check_grad(wide[:, 3 : 3 + d], grad[:, :d], ids, first=2, base=torch.full((v, d), 5.0, device="cuda"))
    assert bool((wide[:, :3] == 5).all() and (wide[:, 3 + d :] == 5).all())


def test_gradient_same_bits(gpu):
    n, v, d = 40000, 1000, 40
    ids = (torch.rand(n, generator=gen(15), device="cuda") ** 6 * v).long()
    grad = normal(gen(16), n, d)
    a = gpu.embedding_grad(grad, ids, v)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        b = gpu.embedding_grad(grad, ids, v)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    check_grad(a, grad, ids)


def test_gradient_special_values_stay_in_their_rows(gpu):
    grad = torch.ones(64, 16, device="cuda")
    ids = torch.arange(64, device="cuda") % 8
    grad[9, 3], grad[2, 4] = float("nan"), float("inf")
    g = gpu.embedding_grad(grad, ids, 10)
    assert bool(torch.isnan(g[1, 3])) and bool(torch.isinf(g[2, 4])) and int((~torch.isfinite(g)).sum()) == 2
    assert float(g[8:].abs().sum()) == 0


def test_autograd_against_differences(gpu):
    table = normal(gen(17), 30, 20).requires_grad_()
    ids = torch.randint(0, 35, (6, 9), generator=gen(18), device="cuda")
    dy, step = normal(gen(19), 6, 9, 20), normal(gen(20), 30, 20)
    out = gpu.torch_embedding(table, ids, scale=3.0)
    (g,) = torch.autograd.grad(out, table, dy)
    f = lambda t: float((gpu.embedding(t.detach(), ids, scale=3.0).double() * dy.double()).sum())  # noqa: E731
    # linear in the table: the difference is the derivative but for the rounding of the looked-up values
    want = (f(table + step) - f(table - step)) / 2
    size = float((gpu.embedding((table.abs() + step.abs()).detach(), ids, scale=3.0).double() * dy.double().abs()).sum())
    assert abs(float((g.double() * step.double()).sum()) - want) <= 2.0 ** -21 * size


def test_autograd_of_views_and_of_sums(gpu):
    """A table with gaps (its own path on the host), ids with gaps, and a gradient that is one number broadcast."""
    base = normal(gen(22), 30, 40)
    ids = torch.randint(0, 30, (6, 10), generator=gen(23), device="cuda")
    grads = []
    for table, at in ((base[:, ::2].contiguous(), ids.T.contiguous()), (base[:, ::2], ids.T)):
        table = table.detach().requires_grad_()
        out = gpu.torch_embedding(table, at, scale=2.0)
        grads.append(torch.autograd.grad(out.sum(), table)[0])
    assert torch.equal(*grads)
    count = torch.bincount(ids.reshape(-1), minlength=30).float()
    assert torch.equal(grads[0], 2 * count[:, None].expand(30, 20))
    table = base.clone().requires_grad_()
    (g,) = torch.autograd.grad(gpu.torch_embedding(table, ids).square().sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(gpu):
    table, ids = normal(gen(21), 10, 8), torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        gpu.embedding(table.double(), ids)
    with pytest.raises(TypeError):
        gpu.embedding(table, ids.float())
    with pytest.raises(ValueError):
        gpu.embedding(table[0], ids)
    with pytest.raises(gpu.NDTensorsError):
        gpu.embedding(table, ids.cpu())
    with pytest.raises(ValueError):
        gpu.embedding_grad(table, ids, 10)
    with pytest.raises(ValueError):
        gpu.embedding_grad(table[:4], ids, -1)
    with pytest.raises(ValueError):
        gpu.embedding_grad(table[:4], ids, 10, out=torch.empty(9, 8, device="cuda"))
    with pytest.raises(TypeError):
        gpu.embedding_grad(table[:4], ids, 10, out_dtype=torch.float64)
    lib, p = gpu.get_lib(), table.data_ptr()
    assert lib.ndt_b200_embedding_dev(2, p, 10, 8, 7, ids.data_ptr(), 1, 4, 0, 1.0, p, 8, None) == -1
    assert lib.ndt_b200_embedding_dev(5, p, 10, 8, 8, ids.data_ptr(), 1, 4, 0, 1.0, p, 8, None) == -1
    assert lib.ndt_b200_embedding_dev(2, p, 10, 8, 8, None, 1, 4, 0, 1.0, p, 8, None) == -1
    assert lib.ndt_b200_embedding_grad_dev(2, p, 8, ids.data_ptr(), 1, 4, 10, 8, 0, 1.0, 2, None, 8, 0, None) == -1
    assert lib.ndt_b200_embedding_grad_dev(2, p, 8, ids.data_ptr(), 1, -4, 10, 8, 0, 1.0, 2, p, 8, 0, None) == -1
