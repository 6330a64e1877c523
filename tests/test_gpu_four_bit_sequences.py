"""The operators on a 4-bit cache together, as a serving loop uses them: prompts
appended with their rotation and attended in chunks, forked, decoded token by
token, freed, the pool compacted, decoded on; every output against 64-bit
attention over the values that the sequence's rows stood for when they were
appended, and every stored value against the rotated row."""
from __future__ import annotations

import pytest
import torch

import attend_oracle
import token_oracle

pytestmark = pytest.mark.gpu

HEADS, GROUP, DIM, BLOCK, LAYERS = 2, 3, 96, 16, 2
P_EPS = 2.0 ** -11  # one rounding of a probability to fp16


class Loop:
    """A pool of 4-bit pages with page tables on the device, and the values of each
    sequence's tokens on the host."""

    def __init__(self, ops, dev, slots, seqs, width, seed, dtype):
        self.ops, self.dev, self.dtype = ops, dev, dtype
        self.gen = torch.Generator().manual_seed(seed)
        row = ops.e2m1_row_bytes(HEADS, DIM)
        self.kv = torch.full((LAYERS, 2, slots, BLOCK, row), 0xff, dtype=torch.uint8, device=dev)  # NaN scales
        self.caches = ops.PlaneTable([self.kv[l, p] for p in range(2) for l in range(LAYERS)], 2)
        self.meta = torch.zeros(slots, dtype=torch.uint8, device=dev)
        self.l2p = torch.full((4 * slots,), -1, dtype=torch.int64, device=dev)
        self.p2l = torch.full((slots,), -1, dtype=torch.int64, device=dev)
        self.start = torch.zeros(1, dtype=torch.int64, device=dev)
        self.tables = torch.full((seqs, width), -1, dtype=torch.int64, device=dev)
        self.lens = torch.zeros(seqs, dtype=torch.int64, device=dev)
        self.table = ops.rotary_table(4096, DIM, base=5e5, device=dev)
        self.next_id = 0
        self.text = [[] for _ in range(seqs)]  # per sequence and token: [layer][K, V] rows of bytes

    def pool(self):
        return self.meta, self.l2p, self.p2l, self.tables, self.lens

    def ids(self, x):
        return torch.tensor(x, dtype=torch.int64, device=self.dev)

    def take(self, n):
        slots = self.ops.pop_reusable_slots(self.meta, self.start, self.ids([]), n)
        old = self.p2l[slots]
        new = torch.arange(self.next_id, self.next_id + n, device=self.dev)
        self.next_id += n
        ones = torch.ones(n, dtype=torch.uint8, device=self.dev)
        self.ops.commit_save_metadata(self.l2p, self.p2l, self.meta, old[old >= 0], new, slots, ones, ones)
        return slots

    def run(self, counts):
        """counts[s] new tokens of sequence s: appended and attended in every layer."""
        seqs = sorted(counts)
        mapping, positions = [], []
        for s in seqs:
            n, have = counts[s], len(self.text[s])
            first, last = -(-have // BLOCK), -(-(have + n) // BLOCK)
            if last > first:
                self.tables[s, first:last] = self.take(last - first)
            pos = torch.arange(have, have + n, device=self.dev)
            mapping.append(self.tables[s, pos // BLOCK] * BLOCK + pos % BLOCK)
            positions.append(pos)
            self.lens[s] = have + n
        mapping, positions = torch.cat(mapping), torch.cat(positions)
        rows = mapping.numel()
        offsets = self.ids([0] + [counts[s] for s in seqs]).cumsum(0)
        tables, lens = self.tables[self.ids(seqs)], self.lens[self.ids(seqs)]
        fresh = [[None] * LAYERS for _ in range(rows)]
        for layer in range(LAYERS):
            both = torch.randn((rows, (GROUP + 2) * HEADS, DIM), generator=self.gen).to(self.dtype)
            q, k, v = both.to(self.dev).split([GROUP * HEADS, HEADS, HEADS], 1)
            caches = self.kv[layer, 0], self.kv[layer, 1]
            q = self.ops.append_tokens(k, v, *caches, mapping, positions=positions, table=self.table, query=q,
                                       check=True)
            stored = [c.flatten(0, 1)[mapping].cpu() for c in caches]
            turned, bound = token_oracle.rotate(k.cpu(), positions.cpu(), self.table.cpu())
            token_oracle.check_e2m1(stored[0], turned, bound, 1.0)
            token_oracle.check_e2m1(stored[1], v.cpu().double(), torch.zeros_like(bound), 1.0)
            for c, rows_of in zip(caches, stored):
                got = self.ops.read_tokens(c, mapping, head_dim=DIM, dtype=torch.float32, check=True)
                assert torch.equal(got.cpu().double(), token_oracle.values(rows_of, HEADS, DIM))
            for r in range(rows):
                fresh[r][layer] = (stored[0][r], stored[1][r])
            if layer == 0:
                first_q = q
            else:
                self.check(seqs, counts, layer, q, fresh, caches, tables, lens, offsets)
        self.check(seqs, counts, 0, first_q, fresh, (self.kv[0, 0], self.kv[0, 1]), tables, lens, offsets)
        at = 0
        for s in seqs:
            self.text[s] = self.text[s] + fresh[at:at + counts[s]]
            at += counts[s]

    def check(self, seqs, counts, layer, q, fresh, caches, tables, lens, offsets):
        if max(counts.values()) == 1:
            out = self.ops.attend_step(q, *caches, tables, lens, check=True)
        else:
            out = self.ops.attend_chunk(q, offsets, *caches, tables, lens, check=True)
        key, value, rows, at, new = [], [], [], 0, 0
        for s in seqs:
            text = self.text[s] + fresh[new:new + counts[s]]
            new += counts[s]
            key += [t[layer][0] for t in text]
            value += [t[layer][1] for t in text]
            rows.append(torch.arange(at, at + len(text)))
            at += len(text)
        key, value = (token_oracle.values(torch.stack(x), HEADS, DIM).unsqueeze(1) for x in (key, value))
        lengths = [r.numel() for r in rows]
        want, _, bound, _ = attend_oracle.attention(q.cpu(), key, value, rows, lengths, [counts[s] for s in seqs],
                                                    p_eps=P_EPS)
        bound = bound + max(lengths) * value.abs().max() * 2.0 ** -32  # weights far below the largest: see four_bit_batch
        err = (out.cpu().double() - want).abs()
        assert torch.isfinite(err).all() and (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_loop_on_four_bits(dtype):
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    dev = torch.device("cuda", 0)
    loop = Loop(ops, dev, slots=48, seqs=6, width=12, seed=3, dtype=dtype)
    loop.run({0: 70, 1: 5, 2: 33})
    loop.run({0: 9, 2: 40})  # the next pieces of two prompts
    for _ in range(3):
        loop.run({0: 1, 1: 1, 2: 1})
    # two samples of sequence 0, one of sequence 2
    parents, children = [0, 0, 2], [3, 4, 5]
    fresh = loop.ops.pop_reusable_slots(loop.meta, loop.start, loop.ids([]), 3)
    ids = loop.ids([180, 181, 182])
    ops.fork_sequences(*loop.pool(), loop.ids(parents), loop.ids(children), fresh, ids, loop.caches, check=True)
    for p, c in zip(parents, children):
        loop.text[c] = list(loop.text[p])
    for _ in range(2):
        loop.run({s: 1 for s in range(6)})
    ops.free_sequences(*loop.pool(), loop.ids([0, 1]), BLOCK, discard=True, check=True)
    loop.text[0], loop.text[1] = [], []
    _, live = ops.compact_pages(*loop.pool(), loop.caches, check=True)
    assert int(loop.tables.max()) < live.item()
    loop.run({2: 1, 3: 1, 4: 1, 5: 1})
    # drafted tokens over what was moved, and a new prompt in the freed pages
    loop.run({2: 3, 3: 1, 4: 2})
    loop.run({0: 50})


def test_a_decode_step_of_a_layer_in_a_graph():
    """Append and attention captured once, replayed for the next tokens with lengths, slots and rows changed in place."""
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    dev = torch.device("cuda", 0)
    dtype, seqs, heads, group, dim = torch.bfloat16, 3, 2, 4, 128
    table = ops.rotary_table(256, dim, device=dev)
    row = ops.e2m1_row_bytes(heads, dim)
    caches = [torch.full((24, BLOCK, row), 0xff, dtype=torch.uint8, device=dev) for _ in range(2)]
    tables = torch.randperm(24, generator=torch.Generator().manual_seed(1)).view(seqs, 8).to(dev)
    lens = torch.zeros(seqs, dtype=torch.int64, device=dev)
    both = torch.zeros((seqs, heads * (group + 2), dim), dtype=dtype, device=dev)
    q, k, v = both.split([heads * group, heads, heads], 1)
    positions, slots = torch.zeros_like(lens), torch.zeros_like(lens)
    turned, out = (torch.empty((seqs, heads * group, dim), dtype=dtype, device=dev) for _ in range(2))

    def layer():
        ops.append_tokens(k, v, *caches, slots, positions=positions, table=table, query=q, query_out=turned, check=False)
        return ops.attend_step(turned, *caches, tables, lens, out=out, check=False)

    graph, gen = None, torch.Generator().manual_seed(2)
    for step in range(40):
        both.copy_(torch.randn(both.shape, generator=gen).to(dtype))
        lens += 1
        positions.copy_(lens - 1)
        slots.copy_(tables.gather(1, (positions // BLOCK)[:, None])[:, 0] * BLOCK + positions % BLOCK)
        if step == 0:
            layer()
        elif step == 1:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                layer()
        if graph is not None:
            graph.replay()
        torch.cuda.synchronize()
        ops.check_status(dev)
        if step % 13:
            continue
        at = torch.arange(step + 1, device=dev)
        rows = [tables[s, at // BLOCK] * BLOCK + at % BLOCK for s in range(seqs)]
        key, value = (token_oracle.values(c.flatten(0, 1)[torch.cat(rows)].cpu(), heads, dim).unsqueeze(1) for c in caches)
        each = [torch.arange(s * (step + 1), (s + 1) * (step + 1)) for s in range(seqs)]
        want, _, bound, _ = attend_oracle.attention(turned.cpu(), key, value, each, [step + 1] * seqs, [1] * seqs,
                                                    p_eps=P_EPS)
        bound = bound + (step + 1) * value.abs().max() * 2.0 ** -32
        assert ((out.cpu().double() - want).abs() <= bound).all()
