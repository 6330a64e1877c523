"""attend_step over 4-bit caches against 64-bit attention over the values that
the rows stand for: head dims, heads, lengths, blocks, layouts, windows, scales,
values that are no numbers, streams and graphs."""
from __future__ import annotations

import math

import pytest
import torch

import attend_oracle
from four_bit_batch import Batch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
P_EPS = 2.0 ** -11  # one rounding of a probability to fp16


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def run(ops, dev, b, **kw):
    key, value = b.on(dev)
    out = torch.full(b.query.shape, 77.0, dtype=b.query.dtype, device=dev)
    lse = torch.full(b.query.shape[:2], 77.0, device=dev)
    got = ops.attend_step(b.query.to(dev), key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev),
                          window=b.window, sinks=b.sinks, out=out, lse=lse, check=True, **b.scales, **kw)
    assert got is out
    return out.cpu().double(), lse.cpu().double()


def check(b, out, lse, **kw):
    rows, (want, want_lse, bound, lse_bound) = b.expect(P_EPS, **kw)
    for s, n in enumerate(b.lens):
        if n == 0:
            assert (out[s] == 0).all() and (lse[s] == -math.inf).all()
        elif n < 0:
            assert (out[s] == 77).all() and (lse[s] == 77).all()
    err = (out[rows] - want).abs()
    assert torch.isfinite(err).all() and (err <= bound).all(), (err / bound).max()
    err = (lse[rows] - want_lse).abs()
    assert torch.isfinite(err).all() and (err <= lse_bound).all(), (err / lse_bound).max()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[1], [16], [17, 0, 1, -1, 33], [300, 15, 129, 64, 500]])
def test_lengths(ops, dev, dtype, lens):
    b = Batch(lens=lens, heads=2, group=4, dim=128, block=16, dtype=dtype, seed=len(lens))
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("heads", [1, 2, 3])
def test_head_dims(ops, dev, dtype, dim, heads):
    b = Batch(lens=[70, 5, 211], heads=heads, group=3, dim=dim, block=16, dtype=dtype, seed=dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (8, 4), (1, 8), (2, 9), (1, 16), (1, 17), (5, 7), (2, 40)])
def test_heads(ops, dev, dim, heads, group):
    b = Batch(lens=[97, 31], heads=heads, group=group, dim=dim, block=16, dtype=BF16, seed=group)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("dim", [160, 256])
def test_groups_of_wide_heads(ops, dev, group, dim):
    b = Batch(lens=[97, 31], heads=2, group=group, dim=dim, block=16, dtype=F16, seed=3)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("block", [1, 2, 5, 16, 24, 48, 64, 257])
@pytest.mark.parametrize("layout", ["nhd", "merged", "apart"])
def test_blocks_and_layouts(ops, dev, block, layout):
    b = Batch(lens=[100, 256, 259, 7], heads=2, group=2, dim=64, block=block, dtype=BF16, layout=layout, seed=block)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (16, 4), (33, 17), (100, 200), (250, 3), (1000, 5)])
def test_windows(ops, dev, dim, window, sinks):
    b = Batch(lens=[1, 17, 101, 250, 411, 0], heads=1, group=8, dim=dim, block=16, dtype=F16, window=window,
              sinks=sinks, seed=window)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("factors", [(0.0625, 0.25), (7.3, 100.0)])
@pytest.mark.parametrize("scale", [None, -0.3, 0.0])
def test_factors_and_scales(ops, dev, factors, scale):
    b = Batch(lens=[40, 90, 3], heads=2, group=4, dim=128, block=16, dtype=BF16, factors=factors, seed=9)
    kw = {} if scale is None else dict(scale=scale)
    check(b, *run(ops, dev, b, **kw), **kw)


def test_large_scores(ops, dev):
    # scores of some hundreds: every exponential but a few underflows
    b = Batch(lens=[130, 33], heads=1, group=4, dim=64, block=16, dtype=BF16, seed=5, magnitude=60.0)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [64, 128, 160])
def test_shared_segments(ops, dev, dim):
    # few long sequences: every one is cut into many runs
    b = Batch(lens=[6000, 1, 2345], heads=1, group=5, dim=dim, block=64, dtype=F16, seed=6)
    check(b, *run(ops, dev, b))


def test_many_sequences(ops, dev):
    b = Batch(lens=attend_oracle.random_lens(7, 1100, 40), heads=1, group=2, dim=32, block=8, dtype=BF16, seed=7)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("side", ["key", "value"])
def test_a_seen_scale_that_is_no_number(ops, dev, side):
    b = Batch(lens=[50, 50], heads=2, group=3, dim=128, block=16, dtype=F16, seed=8)
    rows = b.rows[0 if side == "key" else 1]
    rows[b.tables[0, 1], 3, 2 * 64 + 8 + 2] = 0x7f  # sequence 0, token 19, head 1, dims 32-47
    out, lse = run(ops, dev, b)
    hit = torch.zeros((2, 6, 128), dtype=torch.bool)
    if side == "key":
        hit[0, 3:] = True
    else:
        hit[0, 3:, 32:48] = True
    assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()
    _, (want, _, bound, _) = b.expect(P_EPS)
    assert ((out - want).abs() <= bound)[~hit].all()
    assert torch.isfinite(lse).all() == (side == "value")


def test_out_may_be_the_query(ops, dev):
    b = Batch(lens=[77, 20], heads=2, group=4, dim=64, block=16, dtype=BF16, seed=10)
    key, value = b.on(dev)
    q = b.query.to(dev)
    lens = torch.tensor(b.lens, device=dev)
    want = ops.attend_step(q, key, value, b.tables.to(dev), lens, check=True)
    got = ops.attend_step(q, key, value, b.tables.to(dev), lens, out=q, check=True)
    assert got is q and torch.equal(got, want)


def test_bad_pages_and_lengths(ops, dev):
    b = Batch(lens=[40, 40], heads=1, group=1, dim=64, block=16, dtype=F16, seed=11)
    key, value = b.on(dev)
    tables, lens = b.tables.to(dev), torch.tensor(b.lens, device=dev)
    good = ops.attend_step(b.query.to(dev), key, value, tables, lens, check=True)
    tables[0, 1] = 1 << 40
    out = torch.empty_like(good)
    with pytest.raises(IndexError):
        ops.attend_step(b.query.to(dev), key, value, tables, lens, out=out, check=True)
    assert torch.equal(out[1], good[1])
    tables[0, 1] = b.tables[0, 1]
    lens[0] = 1 << 40
    with pytest.raises(IndexError):
        ops.attend_step(b.query.to(dev), key, value, tables, lens, out=out, check=True)
    assert torch.equal(out[1], good[1])


def test_streams_and_graphs(ops, dev):
    b = Batch(lens=[900, 40, 333], heads=2, group=4, dim=128, block=16, dtype=BF16, seed=12)
    key, value = b.on(dev)
    tables, lens, q = b.tables.to(dev), torch.tensor(b.lens, device=dev), b.query.to(dev)
    want = ops.attend_step(q, key, value, tables, lens, check=True)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = ops.attend_step(q, key, value, tables, lens, check=False)
    side.synchronize()
    assert torch.equal(got, want)
    graph, live = torch.cuda.CUDAGraph(), q.clone()
    with torch.cuda.graph(graph):
        out = ops.attend_step(live, key, value, tables, lens, check=False)
    for factor in (1.0, -0.5):
        live.copy_(q * factor)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attend_step(live, key, value, tables, lens, check=True))


def test_a_cache_past_four_gigabytes(ops, dev):
    heads, dim, block = 8, 128, 16
    slots = (1 << 32) // (576 * block) + 3
    b = Batch(lens=[33], heads=heads, group=2, dim=dim, block=block, dtype=F16, seed=13)
    planes = [torch.empty((slots, block, 576), dtype=torch.uint8, device=dev) for _ in range(2)]
    tables = torch.tensor([[slots - 1, 1, slots - 2]], device=dev)
    for plane, rows in zip(planes, b.rows):
        for col in range(3):
            plane[tables[0, col]] = rows[b.tables[0, col]].to(dev)
    got = ops.attend_step(b.query.to(dev), *planes, tables, torch.tensor([33], device=dev), check=True)
    _, (want, _, bound, _) = b.expect(P_EPS)
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_refusals(ops, dev):
    q = torch.zeros((1, 4, 64), dtype=F16, device=dev)
    ids = torch.zeros((1, 2), dtype=torch.int64, device=dev)
    lens = torch.ones(1, dtype=torch.int64, device=dev)
    good = torch.zeros((2, 16, 80), dtype=torch.uint8, device=dev)
    ops.attend_step(q, good, good.clone(), ids, lens, check=True)
    for cache, match in ((good.view(2, 16, 1, 80), "4-bit"), (good[:, :, :64], "no heads"),
                         (torch.zeros((2, 16, 288), dtype=torch.uint8, device=dev)[:, :, 8:88], "aligned"),
                         (torch.zeros((2, 16, 112), dtype=torch.uint8, device=dev), "multiple of the K/V heads")):
        with pytest.raises(ValueError, match=match):
            ops.attend_step(q, cache, cache.clone() if cache.is_contiguous() else cache, ids, lens)
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.attend_step(q[..., :48].contiguous(), good, good, ids, lens)
