"""A kernel that gave up a wait inside it: the next call reports it, whichever
operator and whichever path through the host that call takes.  The wait here is
one that nothing ends, with a limit of a few microseconds."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def give_up(gpu):
    assert gpu.get_lib().ndt_b200_give_up_wait(20000, None) == 0
    torch.cuda.synchronize()


def calls(gpu):
    x, w = normal(1, 16, 256), normal(2, 48, 256)
    ids = torch.arange(16, device="cuda")
    w8, ws = gpu.quantize_blocks(w, block_rows=128)
    x8, xs = gpu.quantize_blocks(x)
    gaps = x.repeat_interleave(2, 1)[:, ::2]
    h = normal(3, 4, 64).half()
    return {
        "embedding": lambda: gpu.embedding(x, ids),
        "embedding, gaps": lambda: gpu.embedding(gaps, ids),
        "embedding_grad": lambda: gpu.embedding_grad(x, ids, 16),
        "torch_embedding": lambda: gpu.torch_embedding(x, ids),
        "torch_embedding, gaps": lambda: gpu.torch_embedding(gaps, ids),
        "quantize_blocks": lambda: gpu.quantize_blocks(x)[1],
        "scaled_gemm": lambda: gpu.scaled_gemm(x8, xs, w8, ws),
        "scaled_linear": lambda: gpu.scaled_linear(x, w8, ws),
        "scaled_linear, gaps": lambda: gpu.scaled_linear(x.view(4, 4, 256).transpose(0, 1), w8, ws),
        "torch_scaled_linear": lambda: gpu.torch_scaled_linear(x, w),
        "torch_scaled_linear, gaps": lambda: gpu.torch_scaled_linear(x.view(4, 4, 256).transpose(0, 1), w),
        "expert_layer": lambda: gpu.expert_layer(h, h, h[:, None].expand(4, 2, 64), h[:, :, None], 2)[0],
    }


def test_every_call_reports(gpu):
    for name, call in calls(gpu).items():
        want = call()
        give_up(gpu)
        with pytest.raises(gpu.NDTensorsError, match="gave up"):
            call()
        assert torch.equal(call(), want), name  # once


@pytest.mark.parametrize("gaps", [False, True])
def test_backward_passes_report(gpu, gaps):
    x, w, ids = normal(4, 16, 256), normal(5, 48, 256).requires_grad_(), torch.arange(16, device="cuda")
    x = (x.repeat_interleave(2, 1)[:, ::2] if gaps else x).detach().requires_grad_()
    for y in (gpu.torch_scaled_linear(x.view(4, 4, 256) if gaps else x, w), gpu.torch_embedding(x, ids)):
        give_up(gpu)
        with pytest.raises(gpu.NDTensorsError, match="gave up"):
            torch.autograd.grad(y.sum(), x)


def test_the_text_names_no_single_operator(gpu):
    give_up(gpu)
    with pytest.raises(gpu.NDTensorsError) as e:
        gpu.embedding(normal(6, 3, 8), torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert "scaled product or expert layer" in str(e.value)


def test_refusal_of_the_diagnostic(gpu):
    lib = gpu.get_lib()
    for clocks in (0, -1, 1 << 32):
        assert lib.ndt_b200_give_up_wait(clocks, None) == -1
