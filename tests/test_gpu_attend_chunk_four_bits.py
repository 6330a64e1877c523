"""attend_chunk over 4-bit caches against 64-bit attention over the values that
the rows stand for: head dims, heads, lengths, blocks, layouts, windows, scales,
scales that are no numbers at hidden and seen tokens, streams and graphs."""
from __future__ import annotations

import math

import pytest
import torch

from four_bit_batch import Batch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
P_EPS = 2.0 ** -11  # one rounding of a probability to fp16
LEAST = 2.0 ** -32  # of each value: see four_bit_batch


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def offsets_of(b, dev, first=0):
    return torch.tensor([first] + b.new, device=dev).cumsum(0)


def run(ops, dev, b, **kw):
    key, value = b.on(dev)
    rows, heads, dim = b.query.shape
    # three rows before and two behind the chunks stay as they were
    query = torch.cat([torch.full((3, heads, dim), math.nan, dtype=b.query.dtype), b.query,
                       torch.full((2, heads, dim), math.nan, dtype=b.query.dtype)]).to(dev)
    out = torch.full(query.shape, 77.0, dtype=b.query.dtype, device=dev)
    lse = torch.full((rows + 5, heads), 77.0, device=dev)
    got = ops.attend_chunk(query, offsets_of(b, dev, 3), key, value, b.tables.to(dev),
                           torch.tensor(b.lens, device=dev), window=b.window, sinks=b.sinks, out=out, lse=lse,
                           check=True, **b.scales, **kw)
    assert got is out
    for t in (out, lse):
        assert (t[:3] == 77).all() and (t[rows + 3:] == 77).all()
    return out[3:rows + 3].cpu().double(), lse[3:rows + 3].cpu().double()


def expect(b, **kw):
    from attend_oracle import attention

    out, lse, bound, lse_bound = attention(b.query, b.key, b.value, b.tables.clamp(min=0), b.lens, b.new,
                                           window=b.window, sinks=b.sinks, p_eps=P_EPS, **b.scales, **kw)
    top = b.value.nan_to_num().abs().max().item() * b.scales.get("value_scale", 1.0)
    return out, lse, bound + max(b.lens) * top * LEAST, lse_bound


def check(b, out, lse, rows=slice(None), **kw):
    want, want_lse, bound, lse_bound = expect(b, **kw)
    err = (out - want).abs()[rows]
    assert torch.isfinite(err).all() and (err <= bound[rows]).all(), (err / bound[rows]).max()
    err = (lse - want_lse).abs()[rows]
    assert torch.isfinite(err).all() and (err <= lse_bound[rows]).all(), (err / lse_bound[rows]).max()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([128], [128]), ([7, 300], [7, 2]), ([129, 40, 260], [129, 0, 131]),
                                      ([517, 64, 33, 1], [5, 64, 1, 1])])
def test_lengths(ops, dev, dtype, lens, new):
    b = Batch(lens=lens, new=new, heads=2, group=2, dim=128, block=16, dtype=dtype, seed=len(lens))
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("heads", [1, 2, 3])
def test_head_dims(ops, dev, dtype, dim, heads):
    b = Batch(lens=[150, 20], new=[90, 20], heads=heads, group=3, dim=dim, block=16, dtype=dtype, seed=dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (8, 4), (1, 7), (1, 16), (2, 40), (1, 130), (1, 300)])
def test_heads(ops, dev, heads, group):
    b = Batch(lens=[140, 9], new=[13, 9], heads=heads, group=group, dim=64, block=16, dtype=BF16, seed=group)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("block", [1, 5, 16, 48, 128, 200])
@pytest.mark.parametrize("layout", ["nhd", "merged", "apart"])
def test_blocks_and_layouts(ops, dev, block, layout):
    b = Batch(lens=[200, 131], new=[70, 131], heads=2, group=2, dim=64, block=block, dtype=F16, layout=layout,
              seed=block)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [96, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (33, 4), (100, 17), (130, 300), (1000, 5)])
def test_windows(ops, dev, dim, window, sinks):
    b = Batch(lens=[1, 300, 411, 700], new=[1, 300, 150, 20], heads=1, group=2, dim=dim, block=16, dtype=BF16,
              window=window, sinks=sinks, seed=window)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("factors", [(0.0625, 0.25), (7.3, 100.0)])
@pytest.mark.parametrize("scale", [None, -0.3, 0.0])
def test_factors_and_scales(ops, dev, factors, scale):
    b = Batch(lens=[140, 90], new=[40, 90], heads=2, group=2, dim=128, block=16, dtype=F16, factors=factors, seed=1)
    kw = {} if scale is None else dict(scale=scale)
    check(b, *run(ops, dev, b, **kw), **kw)


@pytest.mark.parametrize("dim", [64, 128])
def test_large_scores(ops, dev, dim):
    b = Batch(lens=[700], new=[300], heads=1, group=1, dim=dim, block=16, dtype=F16, seed=5, magnitude=60.0)
    check(b, *run(ops, dev, b))


def test_long_context(ops, dev):
    b = Batch(lens=[9000, 40], new=[3, 7], heads=2, group=4, dim=128, block=64, dtype=BF16, seed=6)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_scales_that_are_no_numbers(ops, dev, dim, window, sinks):
    """A token that a row does not see, but another of its tile does, may hold anything; one that it sees shows."""
    lens, new = [400, 90], [200, 90]
    b, clean = (Batch(lens=lens, new=new, heads=2, group=2, dim=dim, block=16, dtype=F16, window=window, sinks=sinks,
                      seed=9) for _ in range(2))
    planted = [(0, 260), (0, 399), (1, 45), (0, 20)]  # token 20: seen by all rows alike, or by none
    at = 2 * (dim // 2) + dim // 16 + 1  # head 1, dims 16-31
    for s, t in planted:
        if window and t == 20:
            continue
        b.rows[1][b.tables[s, t // 16], t % 16, at] = 0xff
    out, lse = run(ops, dev, b)
    want, want_lse, bound, lse_bound = expect(clean)
    hit, row = torch.zeros(out.shape, dtype=torch.bool), 0
    for s, (n, fresh) in enumerate(zip(lens, new)):
        for p in range(n - fresh, n):
            seen = [t for q, t in planted if q == s and t <= p and (not window or t > p - window or t < sinks)]
            if [t for t in seen if not (window and t == 20)]:
                hit[row, 2:, 16:32] = True
            row += 1
    assert hit.any() and torch.isnan(out[hit]).all()
    assert ((out - want).abs() <= bound)[~hit].all() and ((lse - want_lse).abs() <= lse_bound).all()


def test_keys_that_are_no_numbers_at_hidden_tokens(ops, dev):
    b, clean = (Batch(lens=[300], new=[100], heads=1, group=2, dim=64, block=16, dtype=BF16, seed=4) for _ in range(2))
    b.rows[0][b.tables[0, 250 // 16], 250 % 16, 32 + 3] = 0x7f
    out, lse = run(ops, dev, b)
    before = torch.arange(100) + 200 < 250
    check(clean, out, lse, rows=before)
    assert torch.isnan(out[~before]).all()


def test_steps_and_chunks_agree(ops, dev):
    b = Batch(lens=[300, 45], new=[1, 1], heads=2, group=4, dim=128, block=16, dtype=F16, seed=7)
    key, value = b.on(dev)
    lens = torch.tensor(b.lens, device=dev)
    step = ops.attend_step(b.query.to(dev), key, value, b.tables.to(dev), lens, check=True)
    chunk = ops.attend_chunk(b.query.to(dev), offsets_of(b, dev), key, value, b.tables.to(dev), lens, check=True)
    assert ((step - chunk).abs().cpu().double() <= 2 * expect(b)[2]).all()


def test_the_same_call_gives_the_same_bits_on_every_stream_and_in_a_graph(ops, dev):
    b = Batch(lens=[1600, 77], new=[400, 3], heads=2, group=4, dim=128, block=16, dtype=F16, seed=8)
    key, value = b.on(dev)
    args = (b.query.to(dev), offsets_of(b, dev), key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev))
    want = ops.attend_chunk(*args, check=True)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = ops.attend_chunk(*args, check=False)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attend_chunk(*args, check=False)
    graph.replay()
    torch.cuda.synchronize()
    ops.check_status(dev)
    assert torch.equal(out, want)


def test_head_dims_above_128_are_refused(ops, dev):
    cache = torch.zeros((2, 16, ops.e2m1_row_bytes(1, 160)), dtype=torch.uint8, device=dev)
    ids = torch.zeros((1, 2), dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="at most 128"):
        ops.attend_chunk(torch.zeros((1, 1, 160), dtype=F16, device=dev), torch.tensor([0, 1], device=dev), cache,
                         cache.clone(), ids, ids[:, 0].contiguous() + 1)
