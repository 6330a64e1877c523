"""The waits of the attention kernels over 4-bit caches: one that runs out (a limit
that ordinary work exceeds) reports KVCA_ERR_DEVICE_TIMEOUT, the kernel ends, and
the next call is as any other."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


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


@pytest.mark.parametrize("which", ["step", "chunk"])
@pytest.mark.parametrize("heads,dim", [(8, 128), (1, 128), (3, 64)])
def test_waits_that_run_out(ops, limit, which, heads, dim):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(dim)
    # contexts that keep every warp waiting for rows of several tiles
    lens, new = [120000, 36000, 80000, 1], [70, 900, 3, 1]
    row, pages = ops.e2m1_row_bytes(heads, dim), 7500
    # codes of any kind, scales about 1
    planes = []
    for _ in range(2):
        rows = torch.randint(0, 256, (pages * len(lens), 16, row), generator=g, device=dev, dtype=torch.uint8)
        rows[:, :, heads * dim // 2:] = 0x38
        planes.append(rows)
    tables = torch.randperm(pages * len(lens), generator=g, device=dev).view(len(lens), -1)
    count = len(lens) if which == "step" else sum(new)
    query = torch.randn((count, heads * 4, dim), generator=g, device=dev).bfloat16()
    lens = torch.tensor(lens, device=dev)
    if which == "step":
        call = lambda: ops.attend_step(query, *planes, tables, lens, check=True)  # noqa: E731
    else:
        offsets = torch.tensor([0] + new, device=dev).cumsum(0)
        call = lambda: ops.attend_chunk(query, offsets, *planes, tables, lens, check=True)  # noqa: E731
    want = call()
    assert limit(0) == 2_000_000_000
    if heads == 8 or which == "chunk":  # (with few heads the rows of a step may be there whenever they are looked for)
        with pytest.raises(RuntimeError, match="bounded device-side wait"):
            call()
    for nanoseconds in (0, 500, 2_000, 5_000, 20_000, 100_000):
        limit(nanoseconds)
        for _ in range(3):
            try:
                got = call()
            except RuntimeError as e:
                assert "bounded device-side wait" in str(e)
            else:
                assert torch.equal(got, want)
    limit(2_000_000_000)
    assert torch.equal(call(), want)
