"""Inputs that torch holds with the negative bit: the stored numbers are the
opposite of the tensor's (the imaginary part of a conjugate is such a view)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def negative(x):
    """x again, stored as -x."""
    v = torch._neg_view(-x)
    assert v.is_neg() and torch.equal(v.clone(), x)
    return v


def same(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    assert len(a) == len(b) and all(torch.equal(p.float(), q.float()) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_inputs(gpu, dtype):
    x, w = normal(1, 40, 272).to(dtype), normal(2, 100, 272).to(dtype)
    ids = torch.arange(40, device="cuda") % 7
    w8, ws = gpu.quantize_blocks(w, block_rows=128)
    x8, xs = gpu.quantize_blocks(x)
    for f, args in [(gpu.quantize_blocks, (x,)), (lambda a: gpu.quantize_blocks(a, 128, transposed=True), (x,)),
                    (lambda a, s: gpu.scaled_linear(a, w8, s), (x, ws)),
                    (lambda s, t: gpu.scaled_gemm(x8, s, w8, t), (xs, ws)), (gpu.torch_scaled_linear, (x, w)),
                    (lambda a: gpu.embedding(a, ids), (x,)), (lambda a: gpu.torch_embedding(a, ids), (x,)),
                    (lambda a: gpu.embedding_grad(a, ids, 7), (x,))]:
        same(f(*map(negative, args)), f(*args))


def test_imaginary_part_of_a_conjugate(gpu):
    z = torch.complex(normal(3, 16, 256), normal(4, 16, 256))
    x = z.conj().imag
    assert x.is_neg()
    q, s = gpu.quantize_blocks(x)
    r, t = gpu.quantize_blocks(-z.imag)
    same((q, s), (r, t))


def test_expert_layer(gpu):
    x, router = normal(5, 6, 64).half(), normal(6, 4, 64).half()
    w_in, w_out = normal(7, 4, 48, 64).half() * 0.2, normal(8, 4, 64, 24).half() * 0.2
    same(gpu.expert_layer(*map(negative, (x, router, w_in, w_out)), 2), gpu.expert_layer(x, router, w_in, w_out, 2))
    one, two = torch.full((4, 1, 1), 0.5, device="cuda"), torch.full((4, 1, 1), 0.25, device="cuda")
    e = lambda a, b: gpu.expert_layer(x, router, w_in.to(E4), w_out.to(E4), 2, in_scales=a, out_scales=b)  # noqa: E731
    same(e(negative(one), negative(two)), e(one, two))


@pytest.mark.parametrize("gaps", [False, True])
def test_gradients(gpu, gaps):
    """A gradient comes with the bit where the loss takes the imaginary part of a conjugate."""
    def grads(neg):
        x, w, table = normal(9, 24, 160), normal(10, 40, 160), normal(11, 12, 40)
        x, table = (t.repeat_interleave(2, 1)[:, ::2] if gaps else t for t in (x, table))
        x, w, table = (t.detach().requires_grad_() for t in (x, w, table))
        f = (lambda t: torch._neg_view(-t)) if neg else (lambda t: t)
        y = gpu.torch_scaled_linear(f(x), f(w)) + gpu.torch_embedding(f(table), torch.arange(24, device="cuda") % 12)
        dy = normal(12, 24, 40)
        return torch.autograd.grad(y, (x, w, table), negative(dy) if neg else dy)

    same(grads(True), grads(False))


def test_results_with_the_bit_are_refused(gpu):
    q, s = gpu.quantize_blocks(normal(13, 8, 128))
    for out in (negative(normal(14, 8, 8)),):
        with pytest.raises(ValueError):
            gpu.scaled_gemm(q, s, q, s, out=out)
        with pytest.raises(ValueError):
            gpu.embedding_grad(normal(15, 4, 8), torch.zeros(4, dtype=torch.int64, device="cuda"), 8, out=out)
