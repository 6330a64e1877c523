"""attend_step over 4-bit caches where a run has only a part of a row's heads (more
K/V heads, or tiles of query heads, than a CTA has warps): codes and scales fetched
apart, several segments of a sequence in one run, runs that begin within a K/V
head's tiles; against 64-bit attention.  And head counts that the warps do not
divide into."""
from __future__ import annotations

import pytest
import torch

import attend_oracle
from four_bit_batch import Batch
from test_gpu_attend_step_four_bits import BF16, F16, P_EPS, check, dev, ops, run  # noqa: F401

pytestmark = pytest.mark.gpu

# (K/V heads, query heads of each, head dim): heads of a run of heads in all
PARTS = [(17, 1, 64),    # 1 of 17: a prime above the 16 warps
         (17, 1, 128), (19, 3, 96),
         (24, 2, 32), (24, 2, 96), (24, 2, 128),  # 12 of 24
         (32, 1, 128),   # 16 of 32, two stages of a ring
         (40, 1, 128),   # 10 of 40
         (20, 3, 64),
         (3, 48, 128),   # 3 tiles of 16 query heads to each of 3: runs of one K/V head's tiles
         (3, 41, 128),   # the last tile half empty
         (7, 20, 96),    # 2 tiles each, 7 of 14 to a run: the second begins in the middle of a K/V head
         (5, 40, 128),   # 3 tiles each, 5 of 15 to a run
         (16, 9, 128),   # 8 warps
         (16, 1, 256),   # 8 of 16
         (9, 2, 256),    # 3 of 9
         (11, 1, 256),   # 1 of 11
         (18, 1, 160), (9, 10, 224)]


@pytest.mark.parametrize("heads,group,dim", PARTS)
@pytest.mark.parametrize("layout", ["nhd", "merged", "apart"])
def test_parts_of_the_heads(ops, dev, heads, group, dim, layout):
    b = Batch(lens=[97, 31, 0, 33, 1, -1, 64], heads=heads, group=group, dim=dim, block=16,
              dtype=BF16 if group % 2 else F16, layout=layout, seed=heads + dim)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("heads,group,dim", [(17, 1, 64), (24, 2, 96), (32, 1, 128), (7, 20, 96), (11, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 17), (250, 3)])
def test_windows(ops, dev, heads, group, dim, window, sinks):
    b = Batch(lens=[17, 300, 411], heads=heads, group=group, dim=dim, block=24, dtype=F16, window=window, sinks=sinks,
              layout="apart", seed=window)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("heads,group,dim", [(17, 1, 64), (24, 2, 128), (3, 41, 128), (5, 40, 128), (9, 2, 256)])
def test_segments_over_many_runs(ops, dev, heads, group, dim):
    b = Batch(lens=[2500, 40, 1111], heads=heads, group=group, dim=dim, block=64, dtype=BF16, seed=heads)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("heads,group,dim", [(17, 1, 32), (20, 1, 64), (7, 20, 96)])
def test_runs_over_many_segments(ops, dev, heads, group, dim):
    b = Batch(lens=attend_oracle.random_lens(heads, 150, 70), heads=heads, group=group, dim=dim, block=8, dtype=F16,
              seed=heads)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("heads", [6, 9, 10, 11, 12, 13, 14, 15, 16])
def test_head_counts(ops, dev, heads, dim):
    b = Batch(lens=[130, 33, 700], heads=heads, group=2, dim=dim, block=16, dtype=BF16, seed=heads)
    check(b, *run(ops, dev, b))


@pytest.mark.parametrize("heads,dim", [(24, 96), (17, 128), (9, 256)])
def test_a_scale_that_is_no_number_and_a_bad_page(ops, dev, heads, dim):
    """They reach the heads, and the sequence, that they belong to, and nothing else."""
    b = Batch(lens=[50, 50, 50], heads=heads, group=2, dim=dim, block=16, dtype=F16, seed=8)
    hit = torch.zeros((3, 2 * heads, dim), dtype=torch.bool)
    for head, token, chunk in ((0, 19, 0), (heads // 2, 33, 1), (heads - 1, 16, dim // 16 - 1)):
        at = heads * dim // 2 + head * (dim // 16) + chunk
        b.rows[1][b.tables[1, token // 16], token % 16, at] = 0x7f
        hit[1, 2 * head:2 * head + 2, 16 * chunk:16 * chunk + 16] = True
    out, lse = run(ops, dev, b)
    _, (want, _, bound, _) = b.expect(P_EPS)
    assert torch.isnan(out[hit]).all() and torch.isfinite(lse).all()
    assert ((out - want).abs() <= bound)[~hit].all()
    tables = b.tables.clone()
    tables[0, 2] = 1 << 40
    key, value = b.on(dev)
    again = torch.empty(out.shape, dtype=F16, device=dev)
    with pytest.raises(IndexError):
        ops.attend_step(b.query.to(dev), key, value, tables.to(dev), torch.tensor(b.lens, device=dev), out=again,
                        check=True)
    good = ~hit
    good[0] = False
    assert torch.equal(again.cpu().double()[good], out[good])


def test_streams_graphs_and_places(ops, dev):
    b = Batch(lens=[900, 40, 333], heads=24, group=2, dim=64, block=16, dtype=BF16, seed=12)
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
    assert torch.equal(ops.attend_step(q, key, value, tables, lens, out=q, check=True), want)
