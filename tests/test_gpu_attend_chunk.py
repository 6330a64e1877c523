"""attend_chunk against 64-bit attention: types, head layouts, chunks from one
token to whole prompts, block sizes, strides, windows with sinks, non-finite
values at hidden tokens, refusals."""
from __future__ import annotations

import math

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
# one rounding of a probability to the type of the product: fp16 2^-11, bf16 2^-8
P_EPS = {F16: 2.0 ** -11, BF16: 2.0 ** -8, E4M3: 2.0 ** -11}
TYPES = [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)]


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def offsets_of(b, dev, first=0):
    at = [first]
    for n in b.new:
        at.append(at[-1] + n)
    return torch.tensor(at, device=dev)


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
    return oracle.attention(b.query, b.key, b.value, b.tables.clamp(min=0), b.lens, b.new, window=b.window,
                            sinks=b.sinks, p_eps=P_EPS[b.key.dtype], **b.scales, **kw)


def check(b, out, lse, rows=slice(None), **kw):
    want, want_lse, bound, lse_bound = expect(b, **kw)
    err = (out - want).abs()[rows]
    assert torch.isfinite(err).all() and (err <= bound[rows]).all(), (err / bound[rows]).max()
    err = (lse - want_lse).abs()[rows]
    assert torch.isfinite(err).all() and (err <= lse_bound[rows]).all(), (err / lse_bound[rows]).max()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("lens,new", [([1], [1]), ([128], [128]), ([7, 300], [7, 2]), ([129, 40, 260], [129, 0, 131]),
                                      ([517, 64, 33, 1], [5, 64, 1, 1])])
def test_lengths(ops, dev, dtype, cache, lens, new):
    b = oracle.Batch(lens=lens, new=new, heads=2, group=2, dim=128, block=16, dtype=dtype, cache=cache, seed=len(lens))
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 112, 128])
def test_head_dims(ops, dev, dtype, cache, dim):
    b = oracle.Batch(lens=[150, 20], new=[90, 20], heads=2, group=3, dim=dim, block=16, dtype=dtype, cache=cache,
                     seed=dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [8, 24, 72, 120])
def test_head_dims_of_eight(ops, dev, dim):
    b = oracle.Batch(lens=[150, 20], new=[90, 20], heads=1, group=3, dim=dim, block=16, dtype=F16, seed=dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (8, 4), (1, 7), (1, 16), (2, 40), (1, 130), (1, 300)])
def test_heads(ops, dev, dtype, cache, heads, group):
    b = oracle.Batch(lens=[140, 9], new=[13, 9], heads=heads, group=group, dim=64, block=16, dtype=dtype, cache=cache,
                     seed=group)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("block", [1, 5, 16, 48, 128, 200])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "merged"])
def test_blocks_and_layouts(ops, dev, block, layout):
    b = oracle.Batch(lens=[200, 131], new=[70, 131], heads=2, group=2, dim=64, block=block, dtype=BF16, layout=layout,
                     seed=block)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (33, 4), (100, 17), (130, 300), (1000, 5)])
def test_windows(ops, dev, dtype, cache, window, sinks):
    b = oracle.Batch(lens=[1, 300, 411, 700], new=[1, 300, 150, 20], heads=1, group=2, dim=64, block=16, dtype=dtype,
                     cache=cache, window=window, sinks=sinks, seed=window)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.02, 1.5])
def test_scale_and_query_slices(ops, dev, scale):
    b = oracle.Batch(lens=[140, 90], new=[40, 90], heads=2, group=2, dim=64, block=16, dtype=F16, seed=1)
    key, value = b.on(dev)
    fused = torch.randn((130, 8, 64)).to(F16).to(dev)  # q, k and v heads of one projection
    q = fused[:, 1:5]
    b.query = q.cpu()
    lse = torch.empty((130, 4), device=dev)
    got = ops.attend_chunk(q, offsets_of(b, dev), key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev),
                           scale=scale, lse=lse, check=True)
    check(b, got.cpu().double(), lse.cpu().double(), scale=scale)


def test_idle_sequences_keep_their_rows(ops, dev):
    b = oracle.Batch(lens=[50, 60], new=[20, 30], heads=1, group=2, dim=64, block=16, dtype=F16, seed=2)
    key, value = b.on(dev)
    out = torch.full(b.query.shape, 77.0, dtype=F16, device=dev)
    ops.attend_chunk(b.query.to(dev), offsets_of(b, dev), key, value, b.tables.to(dev),
                     torch.tensor([-1, 60], device=dev), out=out, check=True)
    assert (out[:20] == 77).all()
    want, _, bound, _ = expect(b)
    assert ((out[20:].cpu().double() - want[20:]).abs() <= bound[20:]).all()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_non_finite_values_at_hidden_tokens(ops, dev, dtype, cache, window, sinks):
    """A token that a row does not see, but another of its tile does, may hold anything."""
    lens, new = [400, 90], [200, 90]
    b = oracle.Batch(lens=lens, new=new, heads=1, group=2, dim=64, block=16, dtype=dtype, cache=cache, window=window,
                     sinks=sinks, seed=9)
    clean = oracle.Batch(lens=lens, new=new, heads=1, group=2, dim=64, block=16, dtype=dtype, cache=cache,
                         window=window, sinks=sinks, seed=9)
    bad = math.nan if cache == E4M3 else math.inf
    planted = [(0, 260), (0, 399), (1, 45)]
    for s, t in planted:
        page = b.tables[s, t // 16]
        b.value[page, t % 16] = torch.full((1, 64), bad).to(cache)
        b.key[page, t % 16] = torch.full((1, 64), math.nan).to(cache)
    out, lse = run(ops, dev, b)
    rows, row = [], 0
    for s, (n, fresh) in enumerate(zip(lens, new)):
        for p in range(n - fresh, n):
            seen = [t for q, t in planted if q == s and t <= p and (not window or t > p - window or t < sinks)]
            if seen:
                assert torch.isnan(out[row]).all()
            else:
                rows.append(row)
            row += 1
    assert len(rows) > 100
    check(clean, out, lse, rows=torch.tensor(rows))


def test_large_scores(ops, dev):
    # scores of some hundreds, growing maxima: outputs are rescaled, most exponentials underflow
    b = oracle.Batch(lens=[700], new=[300], heads=1, group=1, dim=64, block=16, dtype=F16, seed=5, magnitude=60.0)
    check(b, *run(ops, dev, b))


def test_growing_maxima(ops, dev):
    # keys along one direction, longer from token to token: every tile raises the maximum
    b = oracle.Batch(lens=[900], new=[64], heads=1, group=2, dim=64, block=16, dtype=BF16, seed=6)
    for t in range(900):
        page = b.tables[0, t // 16]
        b.key[page, t % 16] = (b.key[page, t % 16].float() + t * 0.02).to(BF16)
    b.query = (b.query.float().abs()).to(BF16)
    check(b, *run(ops, dev, b))


def test_steps_and_chunks_agree(ops, dev):
    b = oracle.Batch(lens=[300, 45], new=[1, 1], heads=2, group=4, dim=128, block=16, dtype=F16, seed=7)
    key, value = b.on(dev)
    lens = torch.tensor(b.lens, device=dev)
    step = ops.attend_step(b.query.to(dev), key, value, b.tables.to(dev), lens, check=True)
    chunk = ops.attend_chunk(b.query.to(dev), offsets_of(b, dev), key, value, b.tables.to(dev), lens, check=True)
    bound = expect(b)[2]
    assert ((step - chunk).abs().cpu().double() <= 2 * bound).all()


def dense(q, k, v, lens, new, group):
    """Causal attention in float64 on the GPU, (rows, heads, dim)."""
    out, row = [], 0
    for s, (n, fresh) in enumerate(zip(lens, new)):
        p = torch.arange(n - fresh, n, device=q.device).view(-1, 1)
        hidden = torch.arange(n, device=q.device) > p
        for h in range(q.shape[1]):
            sc = (q[row:row + fresh, h].double() @ k[s][:, h // group].double().T) * q.shape[2] ** -0.5
            w = torch.softmax(sc.masked_fill(hidden, -math.inf), -1)
            out.append((w @ v[s][:, h // group].double(), w @ v[s][:, h // group].double().abs()))
        row += fresh
    heads = q.shape[1]
    pick = [torch.cat([torch.stack([out[s * heads + h][i] for h in range(heads)], 1) for s in range(len(lens))])
            for i in range(2)]
    return pick


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_prompts(ops, dev, dtype, dim):
    lens, new, heads, group, block = [3001, 1500, 2600], [3001, 700, 1], 2, 3, 16
    g = torch.Generator(device=dev).manual_seed(dim)
    pages = [-(-n // block) for n in lens]
    order = torch.randperm(sum(pages), generator=g, device=dev)
    tables = torch.zeros((3, max(pages)), dtype=torch.int64, device=dev)
    key = torch.randn((sum(pages), block, heads, dim), generator=g, device=dev).to(dtype)
    value = torch.randn((sum(pages), block, heads, dim), generator=g, device=dev).to(dtype)
    at = 0
    for s, n in enumerate(pages):
        tables[s, :n] = order[at:at + n]
        at += n
    query = torch.randn((sum(new), heads * group, dim), generator=g, device=dev).to(dtype)
    offs = torch.tensor([0, 3001, 3701, 3702], device=dev)
    got = ops.attend_chunk(query, offs, key, value, tables, torch.tensor(lens, device=dev), check=True)
    k = [key[tables[s, :pages[s]]].flatten(0, 1)[:n] for s, n in enumerate(lens)]
    v = [value[tables[s, :pages[s]]].flatten(0, 1)[:n] for s, n in enumerate(lens)]
    want, share = dense(query, k, v, lens, new, group)
    eps = torch.finfo(dtype).eps / 2
    # a probability's rounding and the score sums (2^-12 covers them), the result's rounding
    assert ((got.double() - want).abs() <= (P_EPS[dtype] + 2.0 ** -12) * share + eps * 1.01 * want.abs() + 2.0 ** -24).all()
    again = ops.attend_chunk(query, offs, key, value, tables, torch.tensor(lens, device=dev), check=True)
    assert torch.equal(got, again)


def test_bad_offsets_lengths_and_pages_are_reported(ops, dev):
    b = oracle.Batch(lens=[40, 60], new=[10, 20], heads=1, group=2, dim=64, block=16, dtype=F16, seed=6)
    key, value = (t.to(dev) for t in (b.key, b.value))
    q, tables = b.query.to(dev), b.tables.to(dev)
    lens = torch.tensor(b.lens, device=dev)
    for offs, value_ in (([0, 10, 31], 31), ([0, 20, 10], 10), ([-1, 10, 30], 10), ([0, -5, 30], -5)):
        with pytest.raises(IndexError):
            ops.attend_chunk(q, torch.tensor(offs, device=dev), key, value, tables, lens, check=True)
    many = torch.tensor([0, 30, 0, 30, 0, 30, 0, 30, 0], device=dev)  # more rows than there are
    with pytest.raises(IndexError):
        ops.attend_chunk(q, many, key, value, tables[:1].repeat(8, 1), torch.full((8,), 40, device=dev), check=True)
    with pytest.raises(IndexError, match="index 19 "):
        ops.attend_chunk(q, offsets_of(b, dev), key, value, tables, torch.tensor([40, 19], device=dev), check=True)
    bad = b.tables.clone()
    bad[1, 0] = 1 << 40
    with pytest.raises(IndexError):
        ops.attend_chunk(q, offsets_of(b, dev), key, value, bad.to(dev), lens, check=True)
    check(b, *run(ops, dev, b))


def test_captured_graphs_replayed_together(ops, dev):
    batches = [oracle.Batch(lens=[600, 77], new=[100, 3], heads=2, group=4, dim=64, block=16, dtype=F16, seed=s)
               for s in (7, 8)]
    side = torch.cuda.Stream(dev)
    graphs = []
    for b in batches:
        key, value = b.on(dev)
        args = (b.query.to(dev), offsets_of(b, dev), key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev))
        out = torch.zeros(b.query.shape, dtype=F16, device=dev)
        ops.attend_chunk(*args, out=out, check=True)
        torch.cuda.synchronize()
        out.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.attend_chunk(*args, out=out, check=False)
        graphs.append((graph, out, args))
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    ops.check_status(dev)
    for b, (_, out, _) in zip(batches, graphs):
        check(b, out.cpu().double(), expect(b)[1])


def test_no_rows(ops, dev):
    key = torch.zeros((4, 16, 1, 64), dtype=F16, device=dev)
    ids = torch.zeros((2, 3), dtype=torch.int64, device=dev)
    out = ops.attend_chunk(torch.zeros((0, 2, 64), dtype=F16, device=dev), torch.zeros(3, dtype=torch.int64, device=dev),
                           key, key, ids, ids[:, 0].contiguous(), check=True)
    assert out.shape == (0, 2, 64)
    with pytest.raises(ValueError, match="at most 128"):
        wide = torch.zeros((4, 16, 1, 136), dtype=F16, device=dev)
        ops.attend_chunk(torch.zeros((1, 2, 136), dtype=F16, device=dev), torch.tensor([0, 1, 1], device=dev), wide,
                         wide, ids, ids[:, 0].contiguous())
