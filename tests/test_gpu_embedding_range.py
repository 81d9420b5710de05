"""Ids and first ids at the ends of 64 bits: an id below the table's first is
outside, however far below."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

LOW, HIGH = -(2 ** 63), 2 ** 63 - 1


@pytest.mark.parametrize("first,ids,rows", [
    (HIGH - 9, [LOW, LOW + 5, HIGH, HIGH - 9, HIGH - 10, 0, -1], [None, None, 9, 0, None, None, None]),
    (HIGH, [LOW, LOW + 1, HIGH, HIGH - 1], [None, None, 0, None]),
    (LOW, [LOW, LOW + 9, LOW + 10, HIGH, 0], [0, 9, None, None, None])])
def test_ends_of_64_bits(gpu, first, ids, rows):
    table = torch.arange(1, 81, device="cuda", dtype=torch.float32).view(10, 8)
    at = torch.tensor(ids, device="cuda")
    want = torch.stack([torch.zeros(8, device="cuda") if r is None else table[r] for r in rows])
    assert torch.equal(gpu.embedding(table, at, first=first), want)
    g = gpu.embedding_grad(torch.ones(len(ids), 8, device="cuda"), at, 10, first=first)
    count = torch.tensor([float(rows.count(r)) for r in range(10)], device="cuda")
    assert torch.equal(g, count[:, None].expand(10, 8))


@pytest.mark.parametrize("first", [2 ** 40, -(2 ** 40)])
def test_32_bit_ids(gpu, first):
    table = torch.ones(10, 8, device="cuda")
    at = torch.tensor([0, 1, -1, 2 ** 31 - 1, -(2 ** 31)], device="cuda", dtype=torch.int32)
    assert not gpu.embedding(table, at, first=first).any()
    assert not gpu.embedding_grad(torch.ones(5, 8, device="cuda"), at, 10, first=first).any()
