"""Operators whose results carry no gradient refuse inputs that ask for one,
rather than train nothing below them."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def calls(gpu):
    x, w = normal(1, 16, 256), normal(2, 48, 256)
    ids = torch.arange(16, device="cuda")
    w8, ws = gpu.quantize_blocks(w, block_rows=128)
    x8, xs = gpu.quantize_blocks(x)
    h = normal(3, 4, 64).half()
    layer = lambda *t: gpu.expert_layer(*t, 2)[0]  # noqa: E731
    experts = (h, h.clone(), h[:, None].expand(4, 2, 64).contiguous(), h[:, :, None].contiguous())
    return [
        (lambda a: gpu.embedding(a, ids), (x,)),
        (lambda a: gpu.embedding(a[:, ::2], ids), (x,)),
        (lambda a: gpu.scaled_linear(a, w8, ws), (x,)),
        (lambda a, s: gpu.scaled_linear(a[:, ::2].repeat(1, 2), w8, s), (x, ws)),
        (lambda s: gpu.scaled_gemm(x8, s, w8, ws), (xs,)),
        (lambda a: gpu.embedding_grad(a, ids, 16), (x,)),
        (layer, experts),
    ]


def test_inputs_that_require_a_gradient(gpu):
    for f, args in calls(gpu):
        want = f(*args)
        for which in range(len(args)):
            asked = [a.detach().clone().requires_grad_(j == which) for j, a in enumerate(args)]
            with pytest.raises(gpu.NDTensorsError, match="gradient"):
                f(*asked)
            with torch.no_grad():
                assert torch.equal(f(*asked), want)
            assert torch.equal(f(*(a.detach() for a in asked)), want)


def test_forward_mode(gpu):
    for f, args in calls(gpu):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(args[0].detach().clone(), torch.ones_like(args[0]))] + list(args[1:])
            with pytest.raises(gpu.NDTensorsError, match="gradient"):
                f(*dual)


@pytest.mark.parametrize("gaps", [False, True])
def test_forward_mode_of_the_trained_operators(gpu, gaps):
    """They have a backward pass and no forward one; torch says so."""
    x, w, ids = normal(5, 16, 256), normal(6, 48, 128), torch.arange(16, device="cuda")
    x = x[:, ::2] if gaps else x[:, :128].contiguous()
    for f in (lambda a: gpu.torch_embedding(a, ids), lambda a: gpu.torch_scaled_linear(a.unsqueeze(0), w)):
        with forward_ad.dual_level(), pytest.raises(RuntimeError):
            f(forward_ad.make_dual(x, torch.ones_like(x)))


def test_quantised_weights_of_a_trained_layer(gpu):
    """Rounding has no gradient: the 8-bit form of a parameter is a constant."""
    w = normal(4, 32, 128).requires_grad_()
    q, s = gpu.quantize_blocks(w, block_rows=128)
    assert not q.requires_grad and not s.requires_grad
