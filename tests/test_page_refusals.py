"""CPU: what the operators on sequences' pages refuse before any launch, and
the plain pool that the GPU tests compare with."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kv_cache_adapter_b200 import _lib
from page_oracle import random_pool


def pool(**kw):
    p = _lib.PagePool(meta_bits=8, reserved=0, slot_meta=4096, num_slots=8, l2p=8192, num_logical=9, p2l=12288,
                      block_tables=16384, table_stride=4, table_width=4, seq_lens=20480, num_seqs=3, block_size=16)
    for name, x in kw.items():
        setattr(p, name, x)
    return p


def cache(**kw):
    planes = (ctypes.c_uint64 * 1)(1 << 20)
    d = _lib.PagedDesc(plane_ptrs=ctypes.cast(planes, ctypes.POINTER(ctypes.c_uint64)), num_blocks=8, block_size=16,
                       block_stride=4096, row_stride=256, index=None)
    for name, x in kw.items():
        setattr(d, name, x)
    d._keep = planes
    return d


def calls(lib, p, c, work=1 << 40):
    """Return codes of the three operators."""
    big = 4096
    return (lib.kvca_fork_sequences(ctypes.byref(p), big, big, big, big, 2, ctypes.byref(c), 1, 256, big, work, big, None),
            lib.kvca_free_sequences(ctypes.byref(p), big, 2, 0, big, work, big, None),
            lib.kvca_compact_pages(ctypes.byref(p), ctypes.byref(c), 1, 256, big, big, big, work, big, None))


@pytest.mark.parametrize("bad", [dict(meta_bits=7), dict(num_slots=-1), dict(num_logical=-1), dict(table_width=-1),
                                 dict(table_stride=3), dict(num_seqs=-1), dict(block_size=0), dict(slot_meta=None),
                                 dict(p2l=None), dict(l2p=None), dict(block_tables=None), dict(seq_lens=None)],
                         ids=lambda b: ",".join(b))
def test_bad_pools(bad):
    assert calls(_lib.load(), pool(**bad), cache()) == (_lib.KVCA_ERR_BAD_ARGUMENT,) * 3


def test_size_limits():
    lib, limit = _lib.load(), _lib.KVCA_ERR_SIZE_LIMIT
    assert calls(lib, pool(num_slots=1 << 31), cache(num_blocks=1 << 31))[1] == limit
    assert calls(lib, pool(table_width=(1 << 25) + 1, table_stride=1 << 26), cache()) == (limit,) * 3
    big = 4096
    assert lib.kvca_free_sequences(ctypes.byref(pool()), big, 64513, 0, big, 1 << 40, big, None) == limit


def test_bad_caches_and_workspaces():
    lib, bad = _lib.load(), _lib.KVCA_ERR_BAD_ARGUMENT
    for c in (dict(num_blocks=7), dict(block_size=8), dict(row_stride=255), dict(block_stride=4095)):
        got = calls(lib, pool(), cache(**c))
        assert got[0] == got[2] == bad, c
    assert calls(lib, pool(), cache(), work=8) == (bad,) * 3
    assert lib.kvca_fork_workspace_bytes(-1, 4) == 0 and lib.kvca_compact_workspace_bytes(-1) == 0
    assert lib.kvca_fork_workspace_bytes(3, 5) == 256 + 15
    assert lib.kvca_free_workspace_bytes(3, 5) == 256 + 3 * 13
    assert lib.kvca_compact_workspace_bytes(4097) == 256 + 4 * (2 + 2 * 4097)


def test_plain_pool_keeps_its_invariants():
    p = random_pool(0, slots=200, seqs=7, longest=90, block=8, empty=5)
    data = torch.arange(200 * 8).view(1, 200, 8).clone()

    def text(s):
        return [int(data[0, p.tables[s][t // 8], t % 8]) for t in range(p.lens[s])]

    def holders():
        count = [0] * 200
        for s, row in enumerate(p.tables):
            for slot in row[:p.pages(s)]:
                count[slot] += 1
        return count

    before = [text(s) for s in range(7)]
    p.fork([0, 1], [8, 9], p.spare[:2], p.unused_ids[:2], data)
    assert text(8) == before[0] and text(9) == before[1] and holders() == p.pin
    p.free([0, 3], True)
    assert holders() == p.pin
    remap, n = p.compact(data)
    assert holders() == p.pin and all(not x for x in p.pin[n:]) and all(x < 0 for x in p.p2l[n:])
    assert [text(s) for s in (1, 2, 4, 5, 6)] == [before[s] for s in (1, 2, 4, 5, 6)] and text(8) == before[0]
    assert all(p.p2l[s] == l for l, s in enumerate(p.l2p) if s >= 0)
