"""Expert layers so wide that fewer than eight tokens fit shared memory beside
the weights' stages: an expert's tokens are taken one to seven at a time, and
the stages shrink to two at the widest."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_experts import check, gen, layer, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", ["bf16", "f16", "f8 bf16", "f8 f16"])
@pytest.mark.parametrize("t,e,top,h,i", [
    (20, 3, 2, 64, 14336), (17, 2, 1, 192, 8192), (20, 3, 2, 320, 6400),
    (17, 2, 2, 64, 5504), (20, 2, 2, 64, 4800), (20, 2, 1, 64, 4200), (30, 2, 2, 7168, 128), (24, 3, 1, 2880, 2880),
    (9, 2, 1, 131, 8191), (9, 2, 2, 72, 14000), (11, 2, 1, 7001, 40), (5, 2, 1, 30000, 64), (5, 2, 1, 29999, 33),
    (3, 2, 2, 64, 15000), (3, 2, 1, 65, 14999), (3, 2, 1, 40000, 16), (3, 2, 1, 39999, 9), (3, 2, 1, 16, 20000),
    (3, 2, 1, 9, 19999), (20, 1, 1, 128, 2688)])
def test_layer(gpu, weights, t, e, top, h, i):
    dtype = torch.bfloat16 if "bf16" in weights else torch.float16
    lay = layer(e, h, i, dtype, "f8" in weights, seed=h + i)
    check(gpu, normal(gen(i), t, h).to(dtype), lay, top, True)


@pytest.mark.parametrize("h,i", [(100000, 8), (8, 50000)])
def test_a_row_that_does_not_fit_is_refused(gpu, h, i):
    router, w_in, w_out, *_ = layer(1, h, i, torch.bfloat16, False)
    with pytest.raises(gpu.NDTensorsError, match="too large"):
        gpu.expert_layer(normal(gen(1), 2, h).to(torch.bfloat16), router, w_in, w_out, 1)
