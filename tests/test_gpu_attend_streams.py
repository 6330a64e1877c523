"""Scratch memory by stream: streams that come back under an old handle, the
per-thread default streams, more streams than counters are kept for."""
from __future__ import annotations

import pytest
import torch

from page_oracle import random_pool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


class Streams:
    """Streams made and destroyed by hand."""

    def __init__(self):
        self.rt = pytest.importorskip("cuda.bindings.runtime")

    def make(self):
        code, stream = self.rt.cudaStreamCreateWithFlags(self.rt.cudaStreamNonBlocking)
        assert int(code) == 0
        return int(stream)

    def destroy(self, stream):
        assert int(self.rt.cudaStreamDestroy(stream)[0]) == 0


def step_args(dev, n=3000):
    g = torch.Generator(device=dev).manual_seed(1)
    kv = torch.randn((2, -(-n // 16) * 2, 16, 1, 64), generator=g, device=dev).half()
    q = torch.randn((2, 4, 64), generator=g, device=dev).half()
    tables = torch.randperm(kv.shape[1], generator=g, device=dev).view(2, -1)
    return q, kv[0], kv[1], tables, torch.tensor([n, n - 7], device=dev)


def test_a_reissued_handle_gets_counters_of_its_own(ops, dev):
    streams = Streams()
    args = step_args(dev)
    want = ops.attend_step(*args, check=True)
    torch.cuda.synchronize()
    seen = {}
    for _ in range(8):
        handle = streams.make()
        with torch.cuda.stream(torch.cuda.ExternalStream(handle, device=dev)):
            got = ops.attend_step(*args, check=False)
            seen.setdefault(handle, []).append(ops._step_counters(dev, handle))
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        streams.destroy(handle)
    again = [c for c in seen.values() if len(c) > 1]
    if not again:
        pytest.skip("no handle came back")
    for counters in again:
        assert len({c.data_ptr() for c in counters}) == len(counters)


def test_many_streams_keep_few_counters(ops, dev):
    streams = Streams()
    args = step_args(dev)
    want = ops.attend_step(*args, check=True)
    torch.cuda.synchronize()
    handles = [streams.make() for _ in range(100)]
    outs = []
    for _ in range(2):
        for handle in handles:
            with torch.cuda.stream(torch.cuda.ExternalStream(handle, device=dev)):
                outs.append(ops.attend_step(*args, check=False))
    torch.cuda.synchronize()
    ops.check_status(dev)
    assert all(torch.equal(out, want) for out in outs)
    assert len(ops._attend_counters) <= 64
    outs.clear()
    for handle in handles:
        streams.destroy(handle)


def test_per_thread_default_streams_are_refused(ops, dev):
    q, key, value, tables, lens = step_args(dev)
    pool = random_pool(1, slots=40, seqs=3, longest=60, block=8)
    planes = [torch.zeros((40, 8, 4), dtype=torch.float16, device=dev)]
    t = pool.tensors(dev)
    offsets = torch.tensor([0, 1, 2], device=dev)
    one = torch.tensor([0], device=dev)
    child = torch.tensor([3], device=dev)
    fresh, ids = torch.tensor(pool.spare[:1], device=dev), torch.tensor(pool.unused_ids[:1], device=dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(2, device=dev)):
        for call in (lambda: ops.attend_step(q, key, value, tables, lens),
                     lambda: ops.attend_chunk(q, offsets, key, value, tables, lens),
                     lambda: ops.fork_sequences(*t, one, child, fresh, ids, planes),
                     lambda: ops.free_sequences(*t, one, 8),
                     lambda: ops.compact_pages(*t, planes)):
            with pytest.raises(ValueError, match="per-thread default stream"):
                call()
    pool.assert_equal(t)
    assert torch.isfinite(ops.attend_step(q, key, value, tables, lens, check=True)).all()
