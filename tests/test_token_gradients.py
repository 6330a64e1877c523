"""CPU: append_tokens refuses a query that wants a gradient, which it would lose."""
from __future__ import annotations

import pytest
import torch

from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops


@pytest.mark.parametrize("in_place", [False, True])
def test_a_query_that_wants_a_gradient(in_place):
    rows = torch.zeros((2, 1, 64), dtype=torch.float16)
    cache = torch.zeros((2, 4, 1, 64), dtype=torch.float16)
    at, table = torch.zeros(2, dtype=torch.int64), ops.rotary_table(4, 64)
    leaf = torch.zeros((2, 2, 64), dtype=torch.float16, requires_grad=True)
    for query in (leaf, leaf * 2):
        call = lambda: ops.append_tokens(rows, rows, cache, cache, at, positions=at, table=table,  # noqa: E731
                                         query=query, query_out=query if in_place else None)
        with pytest.raises(RuntimeError, match="records no gradient"):
            call()
        for off in (torch.no_grad, torch.inference_mode):  # as far as a call without a device comes
            with off(), pytest.raises(ValueError, match="CUDA"):
                call()
    keys = rows.clone().requires_grad_()  # what the cache holds has no graph
    with pytest.raises(ValueError, match="CUDA"):
        ops.append_tokens(keys, keys, cache, cache, at, positions=at, table=table, query=leaf.detach())
