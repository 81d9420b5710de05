"""What a failed call of a language-model operator leaves behind."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_the_next_calls_go_on_after_a_failed_allocation(gpu):
    """The copy of an operand of 2^51 bytes cannot be had; the error is the
    call's alone, not the next kernel launch's of the program."""
    p = torch.zeros(4096, device="cuda")
    a = p.data_ptr()
    rows, k = 2 ** 31 - 4096, 2 ** 20
    data = np.arange(24.0).reshape(2, 3, 4)
    x = gpu.TensorF64.from_numpy(data)
    x.permutedims((2, 0, 1)).to_numpy()

    def fail():
        status = gpu.get_lib().ndt_b200_scaled_gemm_dev(rows, 1, k, 5, a, 0, 1, 128, a, 0, 0, 5, a, 0, 1, 128, a, 0, 0, 2, a, 1,
                                                        0, None)
        assert status == -4 and "memory" in gpu.last_error()

    fail()
    assert np.array_equal(x.permutedims((2, 0, 1)).to_numpy(), data.transpose(2, 0, 1))
    fail()
    assert torch.equal(torch.arange(5, device="cuda").flip(0).cpu(), torch.tensor([4, 3, 2, 1, 0]))
    fail()
    ids = torch.arange(4, device="cuda")
    assert torch.equal(gpu.embedding(p.view(64, 64), ids), p.view(64, 64)[:4])
