"""The language-model operators without a GPU: they resolve from the package,
refuse CPU tensors, and the float64 forms that the GPU tests use agree with
torch's own 8-bit rounding."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from model_ref import experts, quantize, round8, stands_for

NAMES = ["quantize_blocks", "scaled_gemm", "scaled_linear", "torch_scaled_linear", "embedding", "embedding_grad",
         "torch_embedding", "expert_layer"]


@pytest.mark.parametrize("name", NAMES)
def test_resolves_from_the_package(ndt, name):
    assert callable(getattr(ndt, name)) and name in ndt.__all__
    assert getattr(ndt, name).__doc__


def test_unknown_names_are_not_found(ndt):
    with pytest.raises(AttributeError):
        ndt.no_such_operator


def test_no_cpu_path(ndt):
    x, w8, s = torch.ones(4, 128), torch.ones(8, 128).to(torch.float8_e4m3fn), torch.ones(1, 1)
    ids = torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ndt.quantize_blocks(x), lambda: ndt.scaled_gemm(w8, s, w8, s), lambda: ndt.scaled_linear(x, w8, s),
                 lambda: ndt.torch_scaled_linear(x, x), lambda: ndt.embedding(x, ids),
                 lambda: ndt.embedding_grad(x[:3], ids, 4), lambda: ndt.torch_embedding(x, ids),
                 lambda: ndt.expert_layer(x.half(), x.half(), x.half()[:, None], x.half()[:, :, None], 1)):
        with pytest.raises(ndt.NDTensorsError):
            call()


def test_entry_points_fail_without_a_device(ndt):
    if ndt.device_available():
        pytest.skip("a device is present")
    lib = ndt.get_lib()
    assert lib.ndt_b200_embedding_dev(2, None, 1, 1, 1, None, 0, 1, 0, 1.0, None, 1, None) == -4
    assert "embedding" in ndt.last_error() and "no CUDA device" in ndt.last_error()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_round8_is_torchs_rounding(dtype):
    g = torch.Generator().manual_seed(1)
    v = torch.randn(100000, generator=g) * torch.exp(4 * torch.randn(100000, generator=g))
    v = v.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    assert torch.equal(round8(v.double(), dtype), v.to(dtype).double())


def test_quantized_values_are_near(ndt):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(70, 300, generator=g)
    for rows in (1, 128):
        q, s = quantize(x, rows, torch.float8_e4m3fn)
        assert s.shape == (70 if rows == 1 else 1, 3)
        err = (stands_for(q, s, rows) - x.double()).abs()
        # 3 bits of mantissa; below the smallest normal number half a step of 2^-9 scales
        step = s.repeat_interleave(128, 1)[:, :300].repeat_interleave(rows, 0)[:70] * 2.0 ** -10
        assert bool((err <= x.double().abs() * 2.0 ** -4 + step * 1.0001).all())


def test_experts_form_with_one_expert_is_a_gated_layer():
    g = torch.Generator().manual_seed(3)
    x, w_in, w_out = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((4, 6), (1, 10, 6), (1, 6, 5)))
    x = x.to(torch.bfloat16)
    y, ids, weights, bound, _, _ = experts(x, torch.ones(1, 6, dtype=torch.float64), w_in, w_out, 1, False)
    a = x.double() @ w_in[0].T
    assert torch.allclose(y, (torch.nn.functional.silu(a[:, :5]) * a[:, 5:]) @ w_out[0].T)
    assert bool((weights == 1).all()) and bool((ids == 0).all()) and bool((bound > 0).all())
