"""fork_sequences and free_sequences above the size that one block handles:
refusals found late change nothing, duplicates far apart are found; and
compact_pages in graphs."""
from __future__ import annotations

import pytest
import torch

from page_oracle import Pool, random_pool

pytestmark = pytest.mark.gpu

BLOCK, ROW = 4, (4,)


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def wide_pool(bits, *, parents, pages, children):
    """`parents` sequences with `pages` full pages of their own and a partly filled one, then empty ones."""
    per = pages + 1
    slots = parents * per + children + 8
    pool = Pool(slots=slots, logical=slots + children, block=BLOCK, seqs=parents + children, width=per + 1, bits=bits)
    for s in range(parents):
        pool.lens[s] = pages * BLOCK + 1 + s % (BLOCK - 1)
        for k in range(per):
            slot = s * per + k
            pool.tables[s][k], pool.pin[slot], pool.usage[slot] = slot, 1, 3
            pool.p2l[slot], pool.l2p[slot] = slot, slot
    pool.spare = list(range(parents * per, slots))
    pool.unused_ids = list(range(slots, slots + children))
    return pool


class Case:
    """A pool on the device with its cache; `expect` is what it must still be (or have become)."""

    def __init__(self, pool, dev):
        g = torch.Generator().manual_seed(1)
        self.host = torch.randint(-100, 100, (2, pool.slots, BLOCK, *ROW), generator=g).to(torch.float16)
        self.cache = self.host.to(dev)
        self.planes = [self.cache[0], self.cache[1]]
        self.pool, self.dev, self.t = pool, dev, pool.tensors(dev)

    def same(self):
        self.pool.assert_equal(self.t)
        assert torch.equal(self.cache.cpu(), self.host)

    def ids(self, *lists):
        return [torch.tensor(x, dtype=torch.int64, device=self.dev) for x in lists]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("fault", ["unpinned", "outside", "full", "none"])
def test_fork_refused_by_its_last_page(ops, dev, bits, fault):
    """Pages pinned by the blocks that ran before the bad one are unpinned again."""
    pool = wide_pool(bits, parents=12, pages=1500, children=12)
    parents, children = list(range(12)), list(range(12, 24))
    last = pool.tables[11][1499]  # the last full page of the last pair
    error = ValueError
    if fault == "unpinned":
        pool.pin[last] = 0
    elif fault == "outside":
        pool.tables[11][1499], error = pool.slots, IndexError
    elif fault == "full":
        pool.pin[last] = 15 if bits == 8 else 255
    case = Case(pool, dev)
    args = case.ids(parents, children, pool.spare[:12], pool.unused_ids[:12])
    if fault != "none":
        with pytest.raises(error):
            ops.fork_sequences(*case.t, *args, case.planes, check=True)
    else:
        ops.fork_sequences(*case.t, *args, case.planes, check=True)
        pool.fork(parents, children, pool.spare[:12], pool.unused_ids[:12], case.host)
    case.same()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("fault", ["unpinned", "outside", "shared", "none"])
def test_free_refused_by_its_last_page(ops, dev, bits, fault):
    pool = wide_pool(bits, parents=12, pages=1500, children=2)
    last = pool.tables[11][1500]
    error = ValueError
    if fault == "unpinned":
        pool.pin[last] = 0
    elif fault == "outside":
        pool.tables[11][1500], error = 1 << 40, IndexError
    elif fault == "shared":
        pool.tables[11][1500] = pool.tables[0][0]  # pinned once, named by two of the call
    case = Case(pool, dev)
    seqs = list(range(12))
    if fault != "none":
        with pytest.raises(error):
            ops.free_sequences(*case.t, *case.ids(seqs), BLOCK, discard=True, check=True)
    else:
        ops.free_sequences(*case.t, *case.ids(seqs), BLOCK, discard=True, check=True)
        pool.free(seqs, True)
    case.same()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("twice", ["child", "slot", "id", "parent", None])
def test_fork_of_many_sequences(ops, dev, bits, twice):
    """2,500 pairs: the comparison of one block's pairs with another's."""
    n = 2500
    pool = wide_pool(bits, parents=n, pages=2, children=n)
    parents, children = list(range(n)), list(range(n, 2 * n))
    fresh, ids = pool.spare[:n], pool.unused_ids[:n]
    if twice == "child":
        children[2400] = children[7]
    elif twice == "slot":
        fresh[2400] = fresh[7]
    elif twice == "id":
        ids[2400] = ids[7]
    elif twice == "parent":
        parents[2400] = children[7]
    case = Case(pool, dev)
    args = case.ids(parents, children, fresh, ids)
    if twice:
        with pytest.raises(ValueError):
            ops.fork_sequences(*case.t, *args, case.planes, check=True)
    else:
        ops.fork_sequences(*case.t, *args, case.planes, check=True)
        pool.fork(parents, children, fresh, ids, case.host)
    case.same()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("twice", [True, False])
def test_free_of_many_sequences(ops, dev, bits, twice):
    n = 2500
    pool = wide_pool(bits, parents=n, pages=2, children=1)
    seqs = list(range(n))
    if twice:
        seqs[2400] = 7
    case = Case(pool, dev)
    if twice:
        with pytest.raises(ValueError):
            ops.free_sequences(*case.t, *case.ids(seqs), BLOCK, discard=True, check=True)
    else:
        ops.free_sequences(*case.t, *case.ids(seqs), BLOCK, discard=True, check=True)
        pool.free(seqs, True)
    case.same()


@pytest.mark.parametrize("slots", [400, 4096, 20000])
@pytest.mark.parametrize("before", ["copies", "kernel", "nothing"])
def test_compaction_in_a_graph(ops, dev, slots, before):
    """One run of slots (whose first kernel is a programmatic dependent of whatever precedes it) and several."""
    pool = random_pool(slots, slots=slots, seqs=9, longest=slots * BLOCK // 20, block=BLOCK, empty=2)
    case = Case(pool, dev)
    start = [x.clone() for x in case.t]
    bytes_before = case.cache.clone()
    table = ops.PlaneTable(case.planes, 2)
    remap = torch.empty(slots, dtype=torch.int64, device=dev)

    def restore():
        case.cache.copy_(bytes_before)
        for x, s in zip(case.t, start):
            x.copy_(s)

    def work():
        if before != "nothing":
            restore()
        if before == "kernel":
            case.t[4].mul_(1)
        return ops.compact_pages(*case.t, table, remap=remap, check=False)[1]

    restore()
    work()
    torch.cuda.synchronize()
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        live = work()
    for _ in range(3):
        if before == "nothing":
            restore()
        graph.replay()
    torch.cuda.synchronize()
    ops.check_status(dev)
    want, n = pool.compact(case.host)
    assert live.item() == n and remap.tolist() == want
    case.same()
