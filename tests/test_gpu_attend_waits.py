"""The waits of attend_chunk's kernel: one that runs out (a limit that ordinary
work exceeds) reports KVCA_ERR_DEVICE_TIMEOUT, the kernel ends, and the next
call is as any other."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture
def limit(ops):
    """Sets the limit for the test, nanoseconds."""
    lib = ops._lib_handle
    before = lib.kvca_attend_wait_limit(-1)
    yield lib.kvca_attend_wait_limit
    lib.kvca_attend_wait_limit(before)


def prompts(dtype, cache, dim, lens, new):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(dim)
    pages = max(-(-n // 16) for n in lens)
    shape = (pages * len(lens), 16, 4, dim)
    key = torch.randn(shape, generator=g, device=dev).to(cache)
    value = torch.randn(shape, generator=g, device=dev).to(cache)
    query = torch.randn((sum(new), 16, dim), generator=g, device=dev).to(dtype)
    tables = torch.randperm(shape[0], generator=g, device=dev).view(len(lens), -1)
    offsets = torch.tensor([0] + new, device=dev).cumsum(0)
    return query, offsets, key, value, tables, torch.tensor(lens, device=dev)


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (BF16, E4M3)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new", [([3000, 900], [2500, 900]), ([9000] * 12, [3] * 12)])
def test_waits_that_run_out(ops, limit, dtype, cache, dim, lens, new):
    args = prompts(dtype, cache, dim, lens, new)
    want = ops.attend_chunk(*args, check=True)
    assert limit(0) == 2_000_000_000
    with pytest.raises(RuntimeError, match="bounded device-side wait"):
        ops.attend_chunk(*args, check=True)
    # limits that run out at other places, or nowhere
    for nanoseconds in (500, 2_000, 5_000, 20_000, 100_000):
        limit(nanoseconds)
        for _ in range(3):
            try:
                got = ops.attend_chunk(*args, check=True)
            except RuntimeError as e:
                assert "bounded device-side wait" in str(e)
            else:
                assert torch.equal(got, want)
    assert limit(2_000_000_000) == 100_000
    for _ in range(2):
        assert torch.equal(ops.attend_chunk(*args, check=True), want)


def test_the_limit_of_a_graph_is_its_captures(ops, limit):
    args = prompts(F16, F16, 64, [700, 90], [700, 90])
    want = ops.attend_chunk(*args, check=True)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attend_chunk(*args, out=out, check=False)
    limit(0)
    graph.replay()
    torch.cuda.synchronize()
    ops.check_status(torch.device("cuda", 0))
    assert torch.equal(out, want)
