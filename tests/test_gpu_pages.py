"""fork_sequences, free_sequences and compact_pages against plain Python:
metadata of both widths, every plane's bytes, refusals that change nothing."""
from __future__ import annotations

import random

import pytest
import torch

from page_oracle import Pool, random_pool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def make_cache(slots, block, row, planes, dtype, seed, layout="planes"):
    """(CPU copy (planes, slots, block, *row), device tensor, its plane views)."""
    g = torch.Generator().manual_seed(seed)
    host = torch.randint(-100, 100, (planes, slots, block, *row), generator=g).to(dtype)
    if layout == "planes":
        d = host.cuda()
        return host, d, [d[p] for p in range(planes)]
    # merged: (slots, block, planes, *row), token rows of a plane apart from each other
    d = host.permute(1, 2, 0, *range(3, host.dim())).contiguous().cuda()
    return host, d.permute(2, 0, 1, *range(3, host.dim())), [d[:, :, p] for p in range(planes)]


SHAPES = [((2, 8), torch.float16), ((3,), torch.uint8), ((1, 128), torch.bfloat16), ((5,), torch.int16),
          ((3,), torch.int32), ((3,), torch.float64), ((8, 128), torch.float16)]


@pytest.mark.parametrize("row,dtype", SHAPES)
@pytest.mark.parametrize("layout", ["planes", "merged"])
def test_fork_moves_the_last_page(ops, dev, row, dtype, layout):
    pool = random_pool(1, slots=60, seqs=5, longest=70, block=8, empty=6)
    host, cache, planes = make_cache(60, 8, row, 3, dtype, 1, layout)
    t = pool.tensors(dev)
    parents, children = [0, 1, 0, 4], [6, 10, 5, 8]
    fresh, ids = pool.spare[:4], pool.unused_ids[:4]
    ops.fork_sequences(*t, *(torch.tensor(x, device=dev) for x in (parents, children, fresh, ids)), planes, check=True)
    pool.fork(parents, children, fresh, ids, host)
    pool.assert_equal(t)
    assert torch.equal(cache.cpu().double(), host.double())


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("block", [1, 4, 16, 33])
@pytest.mark.parametrize("seed", range(4))
def test_random_programs(ops, dev, bits, block, seed):
    """Forks, frees and compactions one after another."""
    r = random.Random(seed)
    pool = random_pool(seed, slots=400, seqs=9, longest=10 * block, block=block, empty=12, bits=bits,
                       gone=0.2 if seed % 2 else 0.0)
    host, cache, planes = make_cache(400, block, (2, 4), 2, torch.float16, seed)
    t = pool.tensors(dev, stride=len(pool.tables[0]) + 5 if seed == 2 else None)
    for _ in range(12):
        empty = [s for s, n in enumerate(pool.lens) if n == 0]
        full = [s for s, n in enumerate(pool.lens) if n > 0]
        what = r.choice(["fork", "free", "compact"])
        if what == "fork" and empty and full:
            k = r.randint(1, min(4, len(empty)))
            parents, children = [r.choice(full) for _ in range(k)], r.sample(empty, k)
            fresh = r.sample([s for s in range(400) if pool.pin[s] == 0], k)
            ids = r.sample([i for i in range(pool.logical) if pool.l2p[i] < 0], k)
            ops.fork_sequences(*t, *(torch.tensor(x, device=dev) for x in (parents, children, fresh, ids)), planes,
                               check=True)
            pool.fork(parents, children, fresh, ids, host)
        elif what == "free" and full:
            seqs = r.sample(range(len(pool.lens)), r.randint(1, 4))
            discard = r.random() < 0.5
            ops.free_sequences(*t, torch.tensor(seqs, device=dev), block, discard=discard, check=True)
            pool.free(seqs, discard)
        else:
            remap, live = ops.compact_pages(*t, planes, check=True)
            want, n = pool.compact(host)
            assert remap.tolist() == want and live.tolist() == [n]
        pool.assert_equal(t)
        assert torch.equal(cache.cpu(), host)


@pytest.mark.parametrize("bits", [8, 16])
def test_pins_of_shared_pages(ops, dev, bits):
    """Many children of one parent, up to the pin field's maximum and past it."""
    most = 15 if bits == 8 else 255
    pool = Pool(slots=300, logical=400, block=4, seqs=300, width=3, bits=bits)
    pool.tables[0][:2], pool.lens[0] = [7, 9], 8
    pool.pin[7] = pool.pin[9] = 1
    pool.usage[7] = most  # the field next to the pins
    host, cache, planes = make_cache(300, 4, (4,), 1, torch.float16, 0)
    t = pool.tensors(dev)

    def fork(children):
        n = len(children)
        ops.fork_sequences(*t, torch.zeros(n, dtype=torch.int64, device=dev), torch.tensor(children, device=dev),
                           torch.arange(20, 20 + n, device=dev), torch.arange(n, device=dev), planes, check=True)

    with pytest.raises(ValueError):
        fork(list(range(1, most + 1)))  # one too many
    pool.assert_equal(t)
    fork(list(range(1, most)))
    pool.fork([0] * (most - 1), list(range(1, most)), [0] * most, [0] * most, host)
    pool.assert_equal(t)
    with pytest.raises(ValueError):
        fork([299])
    pool.assert_equal(t)
    seqs = list(range(0, most, 2))
    ops.free_sequences(*t, torch.tensor(seqs, device=dev), 4, discard=True, check=True)
    pool.free(seqs, True)
    pool.assert_equal(t)
    rest = list(range(1, most, 2))
    ops.free_sequences(*t, torch.tensor(rest, device=dev), 4, discard=True, check=True)
    pool.free(rest, True)
    pool.assert_equal(t)
    assert pool.pin[7] == 0 and pool.usage[7] == 0


def test_fork_refusals_change_nothing(ops, dev):
    pool = random_pool(3, slots=80, seqs=6, longest=60, block=8, empty=4, shared=False)
    pool.lens[0], pool.lens[1] = 8 * pool.pages(0) - 3, 8 * pool.pages(1)  # a partly filled last page, and none
    assert pool.pages(0) > 1
    host, cache, planes = make_cache(80, 8, (4,), 2, torch.float16, 3)
    free, ids = pool.spare, pool.unused_ids
    mapped = next(l for l in range(pool.logical) if pool.l2p[l] >= 0)
    held = next(s for s in range(80) if pool.pin[s])
    bad = [
        ([99], [6], free[:1], ids[:1], IndexError), ([-1], [6], free[:1], ids[:1], IndexError),
        ([0], [10], free[:1], ids[:1], IndexError), ([0], [6], [80], ids[:1], IndexError),
        ([0], [6], [-1], ids[:1], IndexError), ([0], [6], free[:1], [pool.logical], IndexError),
        ([0], [6], free[:1], [-1], IndexError), ([0], [2], free[:1], ids[:1], ValueError),
        ([0], [0], free[:1], ids[:1], ValueError), ([0, 0], [6, 6], free[:2], ids[:2], ValueError),
        ([0, 6], [6, 7], free[:2], ids[:2], ValueError), ([0], [6], [held], ids[:1], ValueError),
        ([0], [6], free[:1], [mapped], ValueError), ([0, 0], [6, 7], [free[0]] * 2, ids[:2], ValueError),
        ([0, 0], [6, 7], free[:2], [ids[0]] * 2, ValueError),
    ]
    for parents, children, fresh, new, error in bad:
        t = pool.tensors(dev)
        with pytest.raises(error):
            ops.fork_sequences(*t, *(torch.tensor(x, device=dev) for x in (parents, children, fresh, new)), planes,
                               check=True)
        pool.assert_equal(t)
        assert torch.equal(cache.cpu(), host)
    # a page outside the pool, a full page that nobody pinned, a length beyond the table: found after good pages
    for change, error in (("page", IndexError), ("pin", ValueError), ("len", IndexError), ("idle", ValueError)):
        broken = pool.copy()
        if change == "page":
            broken.tables[0][1] = 1 << 33
        elif change == "pin":
            broken.pin[broken.tables[0][1]] = 0
        else:
            broken.lens[0] = 8 * len(broken.tables[0]) + 1 if change == "len" else -3
        t = broken.tensors(dev)
        with pytest.raises(error):
            ops.fork_sequences(*t, *(torch.tensor(x, device=dev) for x in ([1, 0], [7, 6], free[:2], ids[:2])), planes,
                               check=True)
        broken.assert_equal(t)
        assert torch.equal(cache.cpu(), host)
    # unused slots and ids are not looked at
    t = pool.tensors(dev)
    ops.fork_sequences(*t, *(torch.tensor(x, device=dev) for x in ([1, 1], [7, 6], [-5, -5], [-9, -9])), planes,
                       check=True)
    pool.fork([1, 1], [7, 6], [0, 0], [0, 0], host)
    pool.assert_equal(t)


def test_free_refusals_change_nothing(ops, dev):
    pool = random_pool(4, slots=80, seqs=6, longest=60, block=8, empty=2)
    for seqs, error in (([99], IndexError), ([-1], IndexError), ([1, 0, 1], ValueError)):
        t = pool.tensors(dev)
        with pytest.raises(error):
            ops.free_sequences(*t, torch.tensor(seqs, device=dev), 8, check=True)
        pool.assert_equal(t)
    for change, error in (("page", IndexError), ("pin", ValueError), ("len", IndexError)):
        broken = pool.copy()
        if change == "page":
            broken.tables[0][0] = 80
        elif change == "pin":
            broken.pin[broken.tables[0][0]] = 0
        else:
            broken.lens[0] = 8 * len(broken.tables[0]) + 1
        t = broken.tensors(dev)
        with pytest.raises(error):
            ops.free_sequences(*t, torch.tensor([3, 0, 4], device=dev), 8, discard=True, check=True)
        broken.assert_equal(t)
    idle = pool.copy()
    idle.lens[2] = -4
    t = idle.tensors(dev)
    ops.free_sequences(*t, torch.tensor([2, 7], device=dev), 8, discard=True, check=True)
    idle.assert_equal(t)


def test_compact_reports_entries_outside_the_pool(ops, dev):
    pool = random_pool(5, slots=90, seqs=5, longest=60, block=8, empty=1)
    host, cache, planes = make_cache(90, 8, (4,), 1, torch.float16, 5)
    pool.tables[2][0] = 90
    t = pool.tensors(dev)
    with pytest.raises(IndexError, match="index 90 "):
        ops.compact_pages(*t, planes, check=True)
    pool.tables[2][0] = -1
    pool.compact(host)
    pool.tables[2][0] = 90
    pool.assert_equal(t)
    assert torch.equal(cache.cpu(), host)


@pytest.mark.parametrize("slots,live", [(1, 0), (1, 1), (4096, 4096), (4097, 0), (9000, 1), (20000, 12345)])
def test_compact_sizes(ops, dev, slots, live):
    r = random.Random(slots + live)
    pool = Pool(slots=slots, logical=slots, block=1, seqs=1, width=1)
    ids = list(range(slots))
    r.shuffle(ids)
    for s in r.sample(range(slots), live):
        if r.random() < 0.1:
            pool.pin[s] = 1  # pinned, of no logical block
        else:
            pool.p2l[s] = ids.pop()
            pool.l2p[pool.p2l[s]] = s
            pool.usage[s] = r.randint(0, 15)
    host, cache, planes = make_cache(slots, 1, (8,), 2, torch.float16, slots)
    t = pool.tensors(dev)
    remap, n = ops.compact_pages(*t, planes, check=True)
    want, count = pool.compact(host)
    assert n.item() == count == live and remap.tolist() == want
    pool.assert_equal(t)
    assert torch.equal(cache.cpu(), host)


def test_large_fork_and_free(ops, dev):
    pool = random_pool(6, slots=30000, seqs=40, longest=4000, block=8, empty=300, shared=False, resident=0.0)
    host, cache, planes = make_cache(30000, 8, (4,), 1, torch.float16, 6)
    t = pool.tensors(dev)
    parents, children = [j % 40 for j in range(300)], list(range(40, 340))
    fresh, ids = pool.spare[:300], pool.unused_ids[:300]
    ops.fork_sequences(*t, *(torch.tensor(x, device=dev) for x in (parents, children, fresh, ids)), planes, check=True)
    pool.fork(parents, children, fresh, ids, host)
    pool.assert_equal(t)
    assert torch.equal(cache.cpu(), host)
    seqs = list(range(0, 340, 2))
    ops.free_sequences(*t, torch.tensor(seqs, device=dev), 8, discard=True, check=True)
    pool.free(seqs, True)
    pool.assert_equal(t)


def test_graph_replays(ops, dev):
    pool = random_pool(7, slots=200, seqs=6, longest=90, block=8, empty=4)
    host, cache, planes = make_cache(200, 8, (16,), 2, torch.float16, 7)
    t = pool.tensors(dev)
    start = [x.clone() for x in t]
    args = [torch.tensor(x, device=dev) for x in ([0, 3], [7, 6], pool.spare[:2], pool.unused_ids[:2])]
    seqs = torch.tensor([0, 7], device=dev)
    table = ops.PlaneTable(planes, 2)

    def work():
        for x, s in zip(t, start):
            x.copy_(s)
        ops.fork_sequences(*t, *args, table, check=False)
        ops.free_sequences(*t, seqs, 8, discard=True, check=False)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    ops.check_status(dev)
    pool.fork([0, 3], [7, 6], pool.spare[:2], pool.unused_ids[:2], host)
    pool.free([0, 7], True)
    pool.assert_equal(t)
    assert torch.equal(cache.cpu(), host)


def test_argument_checks(ops, dev):
    pool = random_pool(8, slots=20, seqs=2, longest=20, block=8)
    host, cache, planes = make_cache(20, 8, (4,), 1, torch.float16, 8)
    t = list(pool.tensors(dev))
    one = torch.zeros(1, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="same length"):
        ops.fork_sequences(*t, one, one, one, one[:0], planes)
    with pytest.raises(ValueError, match="blocks"):
        ops.fork_sequences(*t, one, one, one, one, [planes[0][:10]])
    with pytest.raises(ValueError, match="block_size"):
        ops.free_sequences(*t, one, 0)
    with pytest.raises(TypeError, match="block_tables"):
        ops.free_sequences(*t[:3], t[3].int(), t[4], one, 8)
    with pytest.raises(ValueError, match="contiguous"):
        ops.compact_pages(*t[:3], t[3].t().contiguous().t(), t[4], planes)
    with pytest.raises(ValueError, match="remap"):
        ops.compact_pages(*t, planes, remap=one)
    with pytest.raises(ValueError, match="slot"):
        ops.free_sequences(t[0], t[1], t[2][:5], t[3], t[4], one, 8)
    ops.fork_sequences(*t, one[:0], one[:0], one[:0], one[:0], planes, check=True)
    ops.free_sequences(*t, one[:0], 8, check=True)
    pool.assert_equal(t)
