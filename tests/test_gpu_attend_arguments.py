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
