"""The example that runs the language-model operators together: its training
step against float64 forms of its products, its decoding step against the plain
form, and its loss."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from model_ref import experts, product_bound, quantize, stands_for

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "language_model.py"
    spec = importlib.util.spec_from_file_location("language_model_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def eight(x, rows):
    return stands_for(*quantize(x, rows, E4), rows)


def test_training_learns(gpu, example):
    table, _, _, _, weight = (p.float() for p in example.make(vocabulary=200, dim=128))
    table.requires_grad_(), weight.requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(1)
    follow = torch.randperm(200, generator=g, device="cuda")
    losses = []
    for _ in range(40):
        ids = torch.randint(0, 200, (512,), generator=g, device="cuda")
        losses.append(float(example.train_step(table, weight, ids, follow[ids], rate=20.0)))
    assert losses[-1] < 0.5 * losses[0] and all(l == l for l in losses)


def test_training_step_is_its_operators(gpu, example):
    """From the logits' own gradient on, the step is the formulas: every
    quantised operand is then known to the bit, and the sums are bounded."""
    table, _, _, _, weight = (p.float() for p in example.make(vocabulary=300, dim=136, seed=2))
    table.requires_grad_(), weight.requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(3)
    ids, targets = (torch.randint(0, 300, (257,), generator=g, device="cuda") for _ in range(2))
    t0, w0 = table.detach().clone(), weight.detach().clone()
    scale = 136 ** 0.5
    hidden = gpu.embedding(t0, ids, scale=scale)
    logits = gpu.torch_scaled_linear(hidden, w0).requires_grad_()
    loss = torch.nn.functional.cross_entropy(logits.float(), targets)
    (d,) = torch.autograd.grad(loss, logits)
    assert torch.equal(example.train_step(table, weight, ids, targets, rate=1.0), loss.detach())
    h8, d8, dt8, ht8, w8 = eight(hidden, 1), eight(d, 1), eight(d.T, 1), eight(hidden.T, 1), eight(w0, 128)
    y = h8 @ w8.T
    assert bool(((logits.detach().double() - y).abs() <= product_bound(h8, w8, y, torch.float32)).all())
    dw, dh = dt8 @ ht8.T, d8 @ w8
    # the products' bounds, and the rounding of the update p - g
    bound = product_bound(dt8, ht8, dw, torch.float32) + 2.0 ** -23 * (w0.double().abs() + dw.abs())
    assert bool((((w0.double() - weight.detach().double()) - dw).abs() <= bound).all())
    zero = torch.zeros_like(t0, dtype=torch.float64)
    dt, size = zero.index_add(0, ids, dh * scale), zero.index_add(0, ids, dh.abs() * scale)
    bound = zero.index_add(0, ids, product_bound(d8, w8.T, dh, torch.float32) * scale)
    bound = bound + 2.0 ** -18 * size + 2.0 ** -23 * (t0.double().abs() + dt.abs())  # (at most 32 rows of an id)
    assert bool((((t0.double() - table.detach().double()) - dt).abs() <= bound).all())


def test_decoding_step(gpu, example):
    table, router, w_in, w_out, weight = example.make(vocabulary=500, dim=256, inner=192, seed=4)
    ids = torch.arange(0, 500, 41, device="cuda")
    decoder = example.Decoder(table, router, w_in, w_out, weight)
    got = decoder.logits(ids)
    x = (table[ids].float() * 16.0).to(torch.bfloat16)
    y = experts(x, router, w_in.double(), w_out.double(), 2, True)[0].to(torch.bfloat16)
    ref = eight(x + y, 1) @ eight(weight, 128).T
    # y may round to the neighbouring bfloat16, and its sum with x to the neighbouring 8-bit number
    assert float((got.double() - ref).norm() / ref.norm()) <= 2e-2
    assert torch.equal(decoder.next_ids(ids), got.argmax(1))
