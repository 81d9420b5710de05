"""The language-model operators inside torch programs that differentiate."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("gaps", [False, True])
def test_results_can_be_changed_in_place(gpu, gaps):
    """y += r on a result of three axes, then the gradients."""
    grads = []
    for in_place in (False, True):
        base, w, r = normal(1, 4, 6, 272), normal(2, 40, 136).requires_grad_(), normal(3, 4, 6, 40).requires_grad_()
        x = (base[..., ::2] if gaps else base[..., :136].contiguous()).detach().requires_grad_()
        y = gpu.torch_scaled_linear(x, w)
        if in_place:
            y += r
        else:
            y = y + r
        grads.append(torch.autograd.grad((y * y).sum(), (x, w, r)))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
