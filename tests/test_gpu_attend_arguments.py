"""Arguments of attend_step and attend_chunk that Python refuses, and results
in the query's place."""
from __future__ import annotations

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def arguments(dev, which, dtype=F16, seed=1):
    lens, new = ([700, 40, 1900], [1, 1, 1]) if which == "step" else ([700, 40, 1900], [300, 40, 7])
    b = oracle.Batch(lens=lens, new=new, heads=2, group=2, dim=64, block=16, dtype=dtype, seed=seed)
    key, value = b.on(dev)
    rest = (key, value, b.tables.to(dev), torch.tensor(lens, device=dev))
    if which == "chunk":
        rest = (torch.tensor([0] + new, device=dev).cumsum(0), *rest)
    return b.query.to(dev), rest


def call_of(ops, which):
    return ops.attend_step if which == "step" else ops.attend_chunk


@pytest.mark.parametrize("which", ["step", "chunk"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (-1, 0), (None, 1), (0, 3), (4, -1), (0.5, 0)])
def test_windows_refused(ops, dev, which, window, sinks):
    query, rest = arguments(dev, which)
    with pytest.raises(ValueError, match="window must be positive"):
        call_of(ops, which)(query, *rest, window=window, sinks=sinks)


@pytest.mark.parametrize("which", ["step", "chunk"])
def test_results_over_other_tensors_refused(ops, dev, which):
    query, rest = arguments(dev, which)
    call, n = call_of(ops, which), query.numel()
    with pytest.raises(TypeError, match="out"):
        call(query, *rest, out=[1.0])
    with pytest.raises(TypeError, match="lse"):
        call(query, *rest, lse=0.0)
    # out begins within the query, and ends there
    both = torch.empty(2 * n, dtype=F16, device=dev)
    row = query.shape[1] * query.shape[2]
    moved = both[:n].view(query.shape).copy_(query)
    with pytest.raises(ValueError, match="out must not overlap query"):
        call(moved, *rest, out=both[row:row + n].view(query.shape))
    moved = both[row:row + n].view(query.shape).copy_(query)
    with pytest.raises(ValueError, match="out must not overlap query"):
        call(moved, *rest, out=both[:n].view(query.shape))
    # the query is every other head of a buffer that begins where out does
    wide = torch.zeros((query.shape[0], 2 * query.shape[1], query.shape[2]), dtype=F16, device=dev)
    with pytest.raises(ValueError, match="out must not overlap query"):
        call(wide[:, ::2], *rest, out=wide.view(-1)[:n].view(query.shape))
    sums = both[:2 * query.shape[0] * query.shape[1]].view(torch.float32).view(query.shape[:2])
    with pytest.raises(ValueError, match="lse must not overlap"):
        call(query, *rest, out=both[:n].view(query.shape), lse=sums)
    with pytest.raises(ValueError, match="lse must not overlap"):
        call(both[:n].view(query.shape), *rest, lse=sums)
    # side by side is fine
    out = both[n:].view(query.shape)
    first = call(query, *rest, check=True)
    assert torch.equal(call(both[:n].view(query.shape).copy_(query), *rest, out=out, check=True), first)


@pytest.mark.parametrize("which", ["step", "chunk"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_result_in_the_query(ops, dev, which, dtype):
    for seed in range(1, 6):
        query, rest = arguments(dev, which, dtype, seed)
        want = call_of(ops, which)(query, *rest, check=True)
        place = query.clone()
        got = call_of(ops, which)(place, *rest, out=place, check=True)
        assert got is place and torch.equal(got, want)
