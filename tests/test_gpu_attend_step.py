"""attend_step against 64-bit attention: types, head layouts, lengths from
none to long ones, block sizes, strides, windows with sinks, refusals."""
from __future__ import annotations

import math

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
# one rounding of a probability: fp16 2^-11; bf16 caches take two bf16 terms, 2^-16 together
P_EPS = {F16: 2.0 ** -11, BF16: 2.0 ** -16, E4M3: 2.0 ** -11}


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def run(ops, dev, b, **kw):
    key, value = b.on(dev)
    rows, heads, dim = b.query.shape
    out = torch.full((rows, heads, dim), 77.0, dtype=b.query.dtype, device=dev)
    lse = torch.full((rows, heads), 77.0, device=dev)
    got = ops.attend_step(b.query.to(dev), key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev),
                          window=b.window, sinks=b.sinks, out=out, lse=lse, check=True, **b.scales, **kw)
    assert got is out
    return out.cpu().double(), lse.cpu().double()


def check(b, out, lse, **kw):
    rows, (want, want_lse, bound, lse_bound) = b.expect(P_EPS[b.key.dtype], **kw)
    for s, n in enumerate(b.lens):
        if n == 0:
            assert (out[s] == 0).all() and (lse[s] == -math.inf).all()
        elif n < 0:
            assert (out[s] == 77).all() and (lse[s] == 77).all()
    err = (out[rows] - want).abs()
    assert torch.isfinite(err).all() and (err <= bound).all(), (err / bound).max()
    err = (lse[rows] - want_lse).abs()
    assert torch.isfinite(err).all() and (err <= lse_bound).all(), (err / lse_bound).max()


TYPES = [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("lens", [[1], [16], [17, 0, 1, -1, 33], [300, 15, 129, 64, 500]])
def test_lengths(ops, dev, dtype, cache, lens):
    b = oracle.Batch(lens=lens, heads=2, group=4, dim=128, block=16, dtype=dtype, cache=cache, seed=len(lens))
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128, 144, 256])
def test_head_dims(ops, dev, dtype, cache, dim):
    b = oracle.Batch(lens=[70, 5, 211], heads=2, group=3, dim=dim, block=16, dtype=dtype, cache=cache, seed=dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [8, 24, 72, 136, 248])
def test_head_dims_of_eight(ops, dev, dim):
    b = oracle.Batch(lens=[70, 5, 211], heads=2, group=3, dim=dim, block=16, dtype=F16, seed=dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (8, 4), (1, 8), (2, 9), (1, 16), (1, 17), (2, 40)])
def test_heads(ops, dev, dtype, cache, heads, group):
    b = oracle.Batch(lens=[97, 31], heads=heads, group=group, dim=64, block=16, dtype=dtype, cache=cache, seed=group)
    check(b, *run(ops, dev, b))


def test_wide_group_at_head_dim_256(ops, dev):
    b = oracle.Batch(lens=[97, 31], heads=1, group=12, dim=256, block=16, dtype=BF16, seed=3)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("block", [1, 2, 5, 16, 24, 48, 64, 257])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "merged"])
def test_blocks_and_layouts(ops, dev, block, layout):
    b = oracle.Batch(lens=[100, 256, 259, 7], heads=2, group=2, dim=64, block=block, dtype=BF16, layout=layout,
                     seed=block)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (16, 4), (33, 17), (100, 200), (250, 3), (1000, 5)])
def test_windows(ops, dev, dtype, cache, window, sinks):
    b = oracle.Batch(lens=[1, 17, 101, 250, 411, 0], heads=1, group=8, dim=64, block=16, dtype=dtype, cache=cache,
                     window=window, sinks=sinks, seed=window)
    check(b, *run(ops, dev, b))


def test_query_slices_and_scale(ops, dev):
    b = oracle.Batch(lens=[40, 90], heads=2, group=2, dim=64, block=16, dtype=F16, seed=1)
    key, value = b.on(dev)
    fused = torch.randn((2, 8, 64)).to(F16).to(dev)  # q, k and v heads of one projection
    q = fused[:, 1:5]
    b.query = q.cpu()
    got = ops.attend_step(q, key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev), scale=-0.3, check=True)
    lse = b.expect(P_EPS[F16], scale=-0.3)[1][1]
    check(b, got.cpu().double(), lse, scale=-0.3)


def test_large_scores_and_negative_infinity_like_values(ops, dev):
    # scores of some hundreds: every exponential but a few underflows
    b = oracle.Batch(lens=[130, 33], heads=1, group=4, dim=64, block=16, dtype=BF16, seed=5, magnitude=60.0)
    check(b, *run(ops, dev, b))


def test_one_long_sequence_over_every_sm(ops, dev):
    n, block = 70_001, 16
    g = torch.Generator(device=dev).manual_seed(3)
    pages = -(-n // block)
    key = torch.randn((pages, block, 1, 64), generator=g, device=dev).to(BF16)
    value = torch.randn((pages, block, 1, 64), generator=g, device=dev).to(BF16)
    query = torch.randn((1, 2, 64), generator=g, device=dev).to(BF16)
    table = torch.randperm(pages, generator=g, device=dev).view(1, -1)
    lse = torch.empty((1, 2), device=dev)
    got = ops.attend_step(query, key, value, table, torch.tensor([n], device=dev), lse=lse, check=True)
    k = key[table[0]].flatten(0, 1)[:n, 0].double()
    v = value[table[0]].flatten(0, 1)[:n, 0].double()
    s = query[0].double() @ k.T / 8
    want = torch.softmax(s, -1) @ v
    # averages of 70,001 values: 2^-16 per probability, the fp32 sums over 1,184 runs, 2^-8 of the result
    share = torch.softmax(s, -1) @ v.abs()
    assert ((got[0].double() - want).abs() <= 2.0 ** -13 * share + 2.0 ** -8 * want.abs()).all()
    assert ((lse[0].double() - torch.logsumexp(s, -1)).abs() <= 2.0 ** -13).all()


def test_many_short_sequences(ops, dev):
    b = oracle.Batch(lens=oracle.random_lens(4, 1500, 21), heads=1, group=2, dim=64, block=8, dtype=F16, seed=4)
    check(b, *run(ops, dev, b))


def test_same_call_twice_gives_the_same_bits(ops, dev):
    b = oracle.Batch(lens=oracle.random_lens(5, 9, 900), heads=2, group=4, dim=128, block=16, dtype=F16, seed=5)
    first, second = run(ops, dev, b), run(ops, dev, b)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])


def test_bad_pages_and_lengths_are_reported(ops, dev):
    b = oracle.Batch(lens=[40, 20], heads=1, group=2, dim=64, block=16, dtype=F16, seed=6)
    key, value = (t.to(dev) for t in (b.key, b.value))
    lens = torch.tensor(b.lens, device=dev)
    q = b.query.to(dev)
    for bad in (-1, b.key.shape[0], 1 << 40):
        tables = b.tables.clone()
        tables[0, 1] = bad
        with pytest.raises(IndexError, match=f"index {bad} "):
            ops.attend_step(q, key, value, tables.to(dev), lens, check=True)
    too_long = 16 * b.tables.shape[1] + 1
    tables = b.tables.clamp(min=0).to(dev)
    with pytest.raises(IndexError, match=f"index {too_long} "):
        ops.attend_step(q, key, value, tables, torch.tensor([too_long, 1], device=dev), check=True)
    check(b, *run(ops, dev, b))  # the device is as before


def test_captured_graphs_replayed_together(ops, dev):
    """Two graphs of the call, captured on one stream and replayed on two, share no workspace."""
    batches = [oracle.Batch(lens=[3000, 77], heads=2, group=4, dim=64, block=16, dtype=F16, seed=s) for s in (7, 8)]
    side = torch.cuda.Stream(dev)
    graphs = []
    for b in batches:
        key, value = b.on(dev)
        args = (b.query.to(dev), key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev))
        out = torch.zeros(b.query.shape, dtype=F16, device=dev)
        ops.attend_step(*args, out=out, check=True)
        torch.cuda.synchronize()
        out.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.attend_step(*args, out=out, check=False)
        graphs.append((graph, out, args))
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for b, (_, out, _) in zip(batches, graphs):
        check(b, out.cpu().double(), b.expect(P_EPS[F16])[1][1])


def test_empty_batch(ops, dev):
    key = torch.zeros((4, 16, 1, 64), dtype=F16, device=dev)
    out = ops.attend_step(torch.zeros((0, 2, 64), dtype=F16, device=dev), key, key,
                          torch.zeros((0, 3), dtype=torch.int64, device=dev),
                          torch.zeros(0, dtype=torch.int64, device=dev), check=True)
    assert out.shape == (0, 2, 64)
