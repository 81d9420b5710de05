"""8-bit block quantisation and block-scaled products against float64 forms.

Quantisation is exact by definition, so it is compared bit for bit.  A product
may differ by the rounding of its 32-bit sums (every one of the k additions
truncated, at worst) and of its result: model_ref.product_bound.
"""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from model_ref import FMAX, product_bound, quantize, stands_for

pytestmark = pytest.mark.gpu

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
REAL = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def same(a, b):
    a, b = a.float().double(), b.double()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


# ------------------------------------------------------------ quantisation


@pytest.mark.parametrize("dtype", REAL)
@pytest.mark.parametrize("q8", [E4, E5])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 129), (128, 128), (130, 260), (257, 4), (5, 1111), (384, 640)])
def test_quantize(gpu, dtype, q8, block_rows, shape):
    x = (normal(gen(1), *shape) * torch.exp(4 * normal(gen(2), shape[0], 1))).to(dtype)
    if dtype == torch.float16:
        x = x.clamp(-60000, 60000)
    q, s, qt, st = gpu.quantize_blocks(x, block_rows, q8, transposed=True)
    rq, rs = quantize(x, block_rows, q8)
    tq, ts = quantize(x.T, block_rows, q8)
    assert q.dtype == q8 and q.shape == x.shape and qt.shape == x.T.shape
    assert torch.equal(s.double(), rs) and same(q, rq)
    assert torch.equal(st.double(), ts) and same(qt, tq)
    # one output alone gives the same
    q1, s1 = gpu.quantize_blocks(x, block_rows, q8)
    t1, u1 = gpu.quantize_blocks(x, block_rows, q8, transposed=True, values=False)
    assert same(q1, rq) and torch.equal(s1, s) and same(t1, tq) and torch.equal(u1, st)


@pytest.mark.parametrize("view", ["transposed", "every other column", "offset", "broadcast"])
def test_quantize_views(gpu, view):
    base = normal(gen(3), 300, 310).to(torch.bfloat16)
    x = {"transposed": base.T, "every other column": base[:, ::2], "offset": base[1:, 3:200],
         "broadcast": base[:1].expand(70, 310)}[view]
    q, s, qt, st = gpu.quantize_blocks(x, transposed=True)
    rq, rs = quantize(x, 1, E4)
    tq, ts = quantize(x.T, 1, E4)
    assert same(q, rq) and torch.equal(s.double(), rs) and same(qt, tq) and torch.equal(st.double(), ts)


@pytest.mark.parametrize("q8", [E4, E5])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(gpu, q8, block_rows):
    x = normal(gen(4), 140, 300)
    x[0] = 0.0
    x[1, :130] = 0.0
    x[2, 5] = float("nan")
    x[3, 7], x[3, 8] = float("inf"), -float("inf")
    x[4] = float("nan")
    x[5] = torch.finfo(torch.float32).max
    x[6] = torch.finfo(torch.float32).min
    x[7] = 2.0 ** -140
    x[8] = 0.0
    x[8, 0] = -2.0 ** -90
    x[9, 128:256] = torch.arange(-64, 64, device="cuda") * 7.0  # ties
    q, s, qt, st = gpu.quantize_blocks(x, block_rows, q8, transposed=True)
    rq, rs = quantize(x, block_rows, q8)
    tq, ts = quantize(x.T, block_rows, q8)
    assert same(q, rq) and torch.equal(s.double(), rs) and same(qt, tq) and torch.equal(st.double(), ts)
    assert torch.isfinite(s).all() and (s > 0).all()


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0)])
def test_quantize_empty(gpu, shape):
    q, s, qt, st = gpu.quantize_blocks(torch.empty(shape, device="cuda"), transposed=True)
    assert q.shape == shape and qt.shape == shape[::-1] and s.shape == (shape[0], -(-shape[1] // 128))


def test_quantize_many_rows(gpu):
    """More rows than a grid's second axis counts, and 64-bit offsets."""
    rows, cols = 2300000, 1000
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.arange(cols, device="cuda")
    x[rows // 2, 5] = -3.0
    q, s = gpu.quantize_blocks(x)
    rq, rs = quantize(x[-1:], 1, E4)
    assert same(q[-1:], rq) and torch.equal(s[-1:].double(), rs)
    assert float(q[rows // 2, 5].float()) == -448 and float(q[: rows // 2].view(torch.uint8).max()) == 0


# ---------------------------------------------------------------- products


def operand(seed, rows, k, block_rows, q8=E4, spread=1.0):
    x = normal(gen(seed), rows, k) * torch.exp(spread * normal(gen(seed + 1), rows, 1))
    q, s = quantize(x, block_rows, q8)
    return q.float().to(q8), s.float(), stands_for(q, s, block_rows)


def check(c, a, b, ref=None):
    ref = a @ b.T if ref is None else ref
    err, bound = (c.double() - ref).abs(), product_bound(a, b, ref, c.dtype)
    assert bool((err <= bound).all()), float((err / bound).max())


SIZES = [(1, 1, 1), (1, 128, 128), (1, 1000, 4096), (7, 300, 640), (128, 128, 128), (129, 257, 385), (64, 2000, 100),
         (200, 520, 16), (300, 1, 2048), (513, 640, 1111), (1000, 1544, 1024), (2500, 2300, 300), (2049, 2049, 129)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("ra,rb", [(1, 128), (1, 1), (128, 128), (128, 1)])
def test_product(gpu, m, n, k, ra, rb):
    a, sa, da = operand(10, m, k, ra)
    b, sb, db = operand(20, n, k, rb)
    for dtype in REAL:
        check(gpu.scaled_gemm(a, sa, b, sb, out_dtype=dtype), da, db)


@pytest.mark.parametrize("ta,tb", [(E4, E5), (E5, E4), (E5, E5)])
@pytest.mark.parametrize("m,n,k", [(33, 200, 300), (2100, 2100, 260)])
def test_product_types(gpu, ta, tb, m, n, k):
    a, sa, da = operand(30, m, k, 1, ta)
    b, sb, db = operand(40, n, k, 1, tb)
    check(gpu.scaled_gemm(a, sa, b, sb, out_dtype=torch.float32), da, db)


@pytest.mark.parametrize("m,n,k", [(5, 130, 700), (140, 140, 140), (2200, 2050, 130)])
@pytest.mark.parametrize("dtype", REAL)
def test_product_accumulates(gpu, m, n, k, dtype):
    a, sa, da = operand(50, m, k, 1)
    b, sb, db = operand(60, n, k, 128)
    c = normal(gen(5), m, n).to(dtype)
    ref = c.double() + da @ db.T
    out = c.clone()
    gpu.scaled_gemm(a, sa, b, sb, out=out, accumulate=True)
    err = (out.double() - ref).abs()
    assert bool((err <= product_bound(da, db, ref, dtype) + 2.0 ** -23 * c.double().abs()).all())


@pytest.mark.parametrize("m,n", [(40, 300), (2100, 2100)])
@pytest.mark.parametrize("view", ["rows apart", "misaligned base", "odd rows", "transposed", "broadcast"])
def test_product_views(gpu, m, n, view):
    """Operands that the tensor maps cannot read in place, and outputs inside wider rows."""
    k = 320
    a, sa, da = operand(70, m, k, 1)
    b, sb, db = operand(80, n, k, 128)

    def moved(q):
        if view == "rows apart":
            wide = torch.zeros(q.shape[0], k + 64, device="cuda").to(E4)
            wide[:, :k] = q
            return wide[:, :k]
        if view == "misaligned base":
            flat = torch.zeros(q.numel() + 3, device="cuda").to(E4)
            flat[3:] = q.reshape(-1)
            return flat[3:].view(q.shape)
        if view == "odd rows":
            wide = torch.zeros(q.shape[0], k + 7, device="cuda").to(E4)
            wide[:, :k] = q
            return wide[:, :k]
        return q.T.contiguous().T if view == "transposed" else q

    if view == "broadcast":
        a, sa, da = a[:1].expand(m, k), sa[:1].expand(m, sa.shape[1]), da[:1].expand(m, k)
    out = torch.full((m, n + 5), 7.0, device="cuda")
    gpu.scaled_gemm(moved(a), sa, moved(b), sb.T.contiguous().T, out=out[:, 1 : n + 1])
    check(out[:, 1 : n + 1], da, db)
    assert bool((out[:, 0] == 7).all() and (out[:, n + 1 :] == 7).all())


def test_product_nan_and_infinity_stay_in_their_rows(gpu):
    a, sa, da = operand(90, 200, 500, 1)
    b, sb, db = operand(95, 300, 500, 128)
    x = a.float()
    x[17, 400] = float("nan")
    a = x.to(E4)
    sa = sa.clone()
    sa[150, 2] = float("inf")
    c = gpu.scaled_gemm(a, sa, b, sb, out_dtype=torch.float32)
    assert bool(torch.isnan(c[17]).all()) and not bool(torch.isfinite(c[150]).any())
    rest = [i for i in range(200) if i not in (17, 150)]
    check(c[rest], da[rest], db)


@pytest.mark.parametrize("m,n,k", [(0, 5, 5), (5, 0, 5), (5, 7, 0)])
def test_product_empty(gpu, m, n, k):
    a, b = torch.zeros(m, k, device="cuda").to(E4), torch.zeros(n, k, device="cuda").to(E4)
    kb = -(-k // 128)
    c = gpu.scaled_gemm(a, torch.ones(m, kb, device="cuda"), b, torch.ones(n, kb, device="cuda"), out_dtype=torch.float32)
    assert c.shape == (m, n) and not c.any()


def test_product_same_bits_twice_and_on_another_stream(gpu):
    a, sa, _ = operand(100, 60, 4000, 1)
    b, sb, _ = operand(110, 1000, 4000, 128)
    c = gpu.scaled_gemm(a, sa, b, sb)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        d = gpu.scaled_gemm(a, sa, b, sb)
    torch.cuda.synchronize()
    assert torch.equal(c, d)


# ------------------------------------------------------------------ layers


@pytest.mark.parametrize("shape,n", [((1, 512), 1000), ((27, 2056), 503), ((2, 3, 130), 64), ((0, 64), 32), ((700, 257), 1600)])
@pytest.mark.parametrize("dtype", REAL)
def test_scaled_linear(gpu, shape, n, dtype):
    x = normal(gen(6), *shape).to(dtype)
    w, sw, dw = operand(120, n, shape[-1], 128)
    y = gpu.scaled_linear(x, w, sw)
    q, s = quantize(x.reshape(-1, shape[-1]), 1, E4)
    assert y.shape == shape[:-1] + (n,) and y.dtype == dtype
    check(y.reshape(-1, n), stands_for(q, s, 1), dw)
    strided = torch.zeros(*shape[:-1], shape[-1] * 2, dtype=dtype, device="cuda")
    strided[..., ::2] = x
    assert torch.equal(gpu.scaled_linear(strided[..., ::2], w, sw), y)


@pytest.mark.parametrize("tokens,n,k", [(1, 8, 8), (64, 136, 200), (1000, 1544, 1111), (300, 129, 5)])
@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                         (torch.float16, torch.float16)])
@pytest.mark.parametrize("grad8", [E4, E5])
def test_gradients_are_the_formulas(gpu, tokens, n, k, dtype, wtype, grad8):
    x = normal(gen(7), tokens, k).to(dtype).requires_grad_()
    w = (normal(gen(8), n, k) * k ** -0.5).to(wtype).requires_grad_()
    dy = normal(gen(9), tokens, n).to(dtype)
    y = gpu.torch_scaled_linear(x, w, grad_dtype=grad8)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == wtype
    vx = lambda m, rows, t=E4: stands_for(*quantize(m.detach(), rows, t), rows)  # noqa: E731
    x8, w8, g8 = vx(x, 1), vx(w, 128), vx(dy, 1, grad8)
    check(y.detach(), x8, w8)
    check(dx, g8, w8.T)
    check(dw, vx(dy.T, 1, grad8), vx(x.T, 1))


@pytest.mark.parametrize("which", ["x", "weight"])
def test_one_gradient_alone(gpu, which):
    x, w = normal(gen(11), 100, 144), normal(gen(12), 80, 144)
    dy = normal(gen(13), 100, 80)
    both = [t.clone().requires_grad_() for t in (x, w)]
    dx, dw = torch.autograd.grad(gpu.torch_scaled_linear(*both), both, dy)
    one = [x.clone().requires_grad_(which == "x"), w.clone().requires_grad_(which == "weight")]
    (d,) = torch.autograd.grad(gpu.torch_scaled_linear(*one), [one[which == "weight"]], dy)
    assert torch.equal(d, dx if which == "x" else dw)


def test_gradients_against_differences(gpu):
    """On values that 8 bits hold exactly the layer is bilinear, so the loss
    sum(dy * y) has exact differences: small integers, every block's largest
    value 448, so each scale is 1 and each operand is its own 8-bit form."""
    tokens, n, k = 130, 150, 140

    def whole(seed, r, c):
        m = torch.randint(-3, 4, (r, c), generator=gen(seed), device="cuda").float()
        m[:, 0::32] = 448.0  # in each block of 1 x 128 of rows ...
        m[0::32, :] = 448.0  # ... and of columns
        return m

    x, w, dy = whole(14, tokens, k), whole(15, n, k), whole(16, tokens, n)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(gpu.torch_scaled_linear(xs, ws), (xs, ws), dy)
    loss = lambda a, b: float((gpu.torch_scaled_linear(a, b).double() * dy.double()).sum())  # noqa: E731
    for t, i, j in [(0, 3, 5), (0, 129, 139), (0, 64, 33), (1, 7, 9), (1, 149, 70), (1, 128, 129)]:
        a, b = x.clone(), w.clone()
        m = (a, b)[t]
        here = float(m[i, j])
        m[i, j] = here + 1 if abs(here) < 4 else here - 32
        step = float(m[i, j]) - here
        got = float((dx, dw)[t][i, j])
        want = (loss(a, b) - loss(x, w)) / step
        # the gradient's own sum, and the rounding of the two losses' row (or column) of y
        bound = 2.0 ** -23 * 160 * float((dy.abs() @ w.abs() if t == 0 else dy.abs().T @ x.abs())[i, j])
        y_err = 2.0 ** -23 * 160 * (x.abs() @ w.abs().T).double() * dy.abs().double()
        far = 2.2 * float((y_err[i] if t == 0 else y_err[:, i]).sum()) / abs(step)
        assert abs(got - want) <= bound + far, (t, i, j, got, want)


def test_gradients_of_views_and_of_sums(gpu):
    """Three axes, x with gaps (its own path on the host), and a gradient that is one number broadcast."""
    base = normal(gen(23), 4, 9, 280)
    w = normal(gen(24), 72, 140)
    grads = []
    for x in (base[..., ::2].contiguous(), base[..., ::2]):
        x, v = x.detach().requires_grad_(), w.clone().requires_grad_()
        y = gpu.torch_scaled_linear(x, v)
        assert y.shape == (4, 9, 72)
        grads.append((y.detach(),) + torch.autograd.grad(y.sum(), (x, v)))
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    x8, ones = base[..., ::2].reshape(36, 140), torch.ones(36, 72, device="cuda")
    vx = lambda m, rows: stands_for(*quantize(m, rows, E4), rows)  # noqa: E731
    check(grads[0][1].view(36, 140), vx(ones, 1), vx(w, 128).T)
    check(grads[0][2], vx(ones.T, 1), vx(x8.T, 1))
    with torch.no_grad():
        assert not gpu.torch_scaled_linear(x, v).requires_grad


def test_gradients_on_another_stream(gpu):
    x, w, dy = normal(gen(25), 64, 256), normal(gen(26), 96, 256), normal(gen(27), 64, 96)
    pairs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            both = [t.clone().requires_grad_() for t in (x, w)]
            pairs.append(torch.autograd.grad(gpu.torch_scaled_linear(*both), both, dy))
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*pairs))


def test_second_derivatives_are_refused(gpu):
    x, w = normal(gen(21), 16, 128).requires_grad_(), normal(gen(22), 16, 128).requires_grad_()
    (dx,) = torch.autograd.grad(gpu.torch_scaled_linear(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# --------------------------------------------------------------- refusals


def test_refusals(gpu):
    a, sa, _ = operand(130, 32, 256, 1)
    b, sb, _ = operand(140, 300, 256, 128)
    x = normal(gen(17), 32, 256)
    err = gpu.NDTensorsError
    with pytest.raises(ValueError):
        gpu.scaled_gemm(a, sa, b[:, :128], sb[:, :1])  # contracted sizes
    with pytest.raises(ValueError):
        gpu.scaled_gemm(a, sa[:, :1], b, sb)  # scales
    with pytest.raises(ValueError):
        gpu.scaled_gemm(a, sa.double(), b, sb)
    with pytest.raises(TypeError):
        gpu.scaled_gemm(x, sa, b, sb)
    with pytest.raises(TypeError):
        gpu.scaled_gemm(a, sa, b, sb, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        gpu.scaled_gemm(a, sa, b, sb, accumulate=True)
    with pytest.raises(ValueError):
        gpu.scaled_gemm(a, sa, b, sb, out=torch.empty(300, 32, device="cuda").T)
    with pytest.raises(err):
        gpu.scaled_gemm(a, sa.cpu(), b, sb)
    with pytest.raises(err):
        gpu.quantize_blocks(x.cpu())
    with pytest.raises(TypeError):
        gpu.quantize_blocks(x.double())
    with pytest.raises(ValueError):
        gpu.quantize_blocks(x, block_rows=64)
    with pytest.raises(ValueError):
        gpu.quantize_blocks(x[0])
    with pytest.raises(ValueError):
        gpu.scaled_linear(x[:, :255], b, sb)
    with pytest.raises(ValueError):
        gpu.scaled_linear(x, b, sb.repeat_interleave(128, 0)[:300])  # scales of single rows
    with pytest.raises(ValueError):
        gpu.torch_scaled_linear(x, normal(gen(18), 5, 255))
    with pytest.raises(TypeError):
        gpu.torch_scaled_linear(x, x, grad_dtype=torch.float16)
    assert FMAX[E4] == torch.finfo(E4).max and FMAX[E5] == torch.finfo(E5).max


def test_c_entry_refusals(gpu):
    lib = gpu.get_lib()
    p = torch.zeros(4096, device="cuda").data_ptr()
    q = lib.ndt_b200_quantize_dev
    assert q(2, p, 4, 4, 4, 1, 1, 5, p + 1024, 16, p + 2048, 1, 4, None, 0, None, 0, 0, None) == 0
    assert q(0, p, 4, 4, 4, 1, 1, 5, p + 1024, 16, p + 2048, 1, 4, None, 0, None, 0, 0, None) == -1  # float64
    assert q(2, p, 4, 4, 4, 1, 1, 5, p + 1024, 15, p + 2048, 1, 4, None, 0, None, 0, 0, None) == -1  # leading dimension
    assert q(2, p, 4, 4, 4, 1, 1, 5, p + 1025, 16, p + 2048, 1, 4, None, 0, None, 0, 0, None) == -1  # base
    assert q(2, p, 4, 4, 4, 1, 2, 5, p + 1024, 16, p + 2048, 1, 4, None, 0, None, 0, 0, None) == -1  # block
    assert q(2, None, 4, 4, 4, 1, 1, 5, p + 1024, 16, p + 2048, 1, 4, None, 0, None, 0, 0, None) == -1
    assert q(2, p, -1, 4, 4, 1, 1, 5, p + 1024, 16, p + 2048, 1, 4, None, 0, None, 0, 0, None) == -1
    assert "quantize" in gpu.last_error()
    gemm = lib.ndt_b200_scaled_gemm_dev
    ok = [4, 4, 16, 5, p, 16, 1, 1, p + 1024, 1, 4, 5, p, 16, 1, 1, p + 1024, 1, 4, 2, p + 4096, 4, 0, None]
    assert gemm(*ok) == 0
    for at, value in [(3, 2), (7, 3), (8, None), (4, None), (19, 5), (20, None), (21, 3), (0, -1)]:
        args = list(ok)
        args[at] = value
        assert gemm(*args) == -1, at
    torch.cuda.synchronize()
