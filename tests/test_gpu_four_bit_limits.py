"""A limit of 0 runs out in the decode step over 4-bit caches of few heads and of parts
of the heads too, where contexts are long; the calls after it are as any other."""
from __future__ import annotations

import pytest
import torch

from test_gpu_four_bit_waits import limit, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,tokens", [(1, 128, 500000), (3, 64, 100000), (17, 128, 100000), (24, 64, 100000)])
def test_a_limit_of_nothing_runs_out(ops, limit, heads, dim, tokens):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(dim)
    row, pages = ops.e2m1_row_bytes(heads, dim), tokens // 16
    planes = []
    for _ in range(2):
        rows = torch.randint(0, 256, (4 * pages, 16, row), generator=g, device=dev, dtype=torch.uint8)
        rows[:, :, heads * dim // 2:] = 0x38
        planes.append(rows)
    tables = torch.randperm(4 * pages, generator=g, device=dev).view(4, -1)
    lens = torch.tensor([16 * pages, 16 * pages - 5, 3, 16 * pages], device=dev)
    query = torch.randn((4, heads * 4, dim), generator=g, device=dev).bfloat16()
    call = lambda: ops.attend_step(query, *planes, tables, lens, check=True)  # noqa: E731
    want = call()
    before, ran_out = limit(0), 0
    for _ in range(10):
        try:
            got = call()
        except RuntimeError as e:
            assert "bounded device-side wait" in str(e)
            ran_out += 1
        else:
            assert torch.equal(got, want)
    assert ran_out > 0
    limit(before)
    for _ in range(3):
        assert torch.equal(call(), want)
