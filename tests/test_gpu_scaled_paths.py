"""Products long enough to go round the kernels' rings of stages and scales,
and the split of k in every form.

The bound is that of the order of the sum: the 128 products of a block, every
addition truncated at worst, then one addition for each block.  That is far
below k additions, so a short accumulator or a missing element shows.
"""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from model_ref import FLOOR, UNIT, quantize, stands_for
from test_gpu_scaled import E4, E5, REAL, gen, normal, operand

pytestmark = pytest.mark.gpu


def check(c, a, b, base=None):
    """c = a b^T (+ base)."""
    k = a.shape[1]
    ref, size = a @ b.T, a.abs() @ b.abs().T
    if base is not None:
        ref, size = ref + base.double(), size + base.double().abs()
    bound = (min(k, 128) + -(-k // 128) + 16) * 2.0 ** -23 * size + UNIT[c.dtype] * 1.01 * ref.abs() + FLOOR[c.dtype]
    err = (c.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


#: CTA pairs over two waves of tiles and several rounds of the ring; one CTA a
#: tile; k split over a cluster with many rows and with few
SIZES = [(2100, 2304, 2056), (2100, 2304, 4100), (1000, 700, 1300), (300, 520, 8200), (130, 140, 33000), (300, 520, 16500), (65, 129, 4096),
         (40, 300, 4100), (17, 1000, 8200), (3, 5000, 2049)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("ra,rb", [(1, 128), (1, 1), (128, 1)])
def test_product(gpu, m, n, k, ra, rb):
    a, sa, da = operand(10, m, k, ra, spread=0.5)
    b, sb, db = operand(20, n, k, rb, spread=0.5)
    first = {}
    for dtype in REAL:
        first[dtype] = gpu.scaled_gemm(a, sa, b, sb, out_dtype=dtype)
        check(first[dtype], da, db)
    assert torch.equal(gpu.scaled_gemm(a, sa, b, sb, out_dtype=torch.float32), first[torch.float32])


@pytest.mark.parametrize("m,n,k", [(2100, 2304, 2056), (300, 520, 8200), (300, 520, 16500), (130, 139, 33000), (40, 300, 4100),
                                   (1000, 701, 1300)])
@pytest.mark.parametrize("dtype", REAL)
def test_accumulates_into_wider_rows(gpu, m, n, k, dtype):
    a, sa, da = operand(30, m, k, 1, spread=0.5)
    b, sb, db = operand(40, n, k, 128, spread=0.5)
    wide = normal(gen(1), m, n + 9).to(dtype) * 8
    before = wide.clone()
    gpu.scaled_gemm(a, sa, b, sb, out=wide[:, 4 : n + 4], accumulate=True)
    check(wide[:, 4 : n + 4], da, db, before[:, 4 : n + 4])
    assert torch.equal(wide[:, :4], before[:, :4]) and torch.equal(wide[:, n + 4 :], before[:, n + 4 :])


@pytest.mark.parametrize("ta,tb", [(E5, E4), (E4, E5)])
@pytest.mark.parametrize("m,n,k", [(2100, 2304, 2056), (300, 520, 8200), (300, 520, 16500), (20, 300, 8200)])
def test_types(gpu, ta, tb, m, n, k):
    a, sa, da = operand(50, m, k, 1, ta)
    b, sb, db = operand(60, n, k, 1, tb)
    check(gpu.scaled_gemm(a, sa, b, sb, out_dtype=torch.float32), da, db)


@pytest.mark.parametrize("tokens,n,k", [(8300, 200, 300), (4097, 129, 2500), (17000, 200, 140)])
def test_gradients_of_many_tokens(gpu, tokens, n, k):
    """The weights' gradient sums over many tokens for few outputs: its k is split."""
    x, w = normal(gen(2), tokens, k).requires_grad_(), (normal(gen(3), n, k) * k ** -0.5).requires_grad_()
    dy = normal(gen(4), tokens, n)
    y = gpu.torch_scaled_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    form = lambda m, rows: stands_for(*quantize(m.detach(), rows, E4), rows)  # noqa: E731
    check(y.detach(), form(x, 1), form(w, 128))
    check(dx, form(dy, 1), form(w, 128).T)
    check(dw, form(dy.T, 1), form(x.T, 1))


def test_one_missing_element_shows(gpu):
    """The bound is tight enough: the same product without one k is outside it."""
    a, sa, da = operand(70, 300, 8200, 1, spread=0.5)
    b, sb, db = operand(80, 520, 8200, 128, spread=0.5)
    c = gpu.scaled_gemm(a, sa, b, sb, out_dtype=torch.float32)
    short = da.clone()
    short[:, 4000] = 0
    with pytest.raises(AssertionError):
        check(c, short, db)
