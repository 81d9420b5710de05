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


def test_results_written_to_out_count_as_changed(gpu):
    """A tensor that a graph has saved, overwritten by a call: its backward pass is refused, not wrong."""
    q, s = gpu.quantize_blocks(normal(4, 8, 128))
    ids = torch.arange(8, device="cuda")
    for write in (lambda c: gpu.scaled_gemm(q, s, q, s, out=c), lambda c: gpu.scaled_gemm(q, s, q, s, out=c, accumulate=True),
                  lambda c: gpu.embedding_grad(normal(5, 8, 8), ids, 8, out=c)):
        p, c = normal(6, 8, 8).requires_grad_(), normal(7, 8, 8)
        loss = (p * c).sum()
        before = c._version
        write(c)
        assert c._version > before
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():
        c = torch.zeros(8, 8, device="cuda")
        gpu.scaled_gemm(q, s, q, s, out=c)
    gpu.scaled_gemm(q, s, q, s, out=c)
    assert bool(c.any())
