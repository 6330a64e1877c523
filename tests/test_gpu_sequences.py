"""The operators on sequences together, as a serving loop uses them: prompts
written and attended in chunks, forked into samples, decoded token by token,
freed, the pool compacted, and decoded on; every output against 64-bit
attention over the tokens that the sequence should hold."""
from __future__ import annotations

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu

LAYERS, HEADS, GROUP, DIM, BLOCK = 2, 2, 3, 64, 16
P_EPS = {"step": 2.0 ** -11, "chunk": 2.0 ** -11}  # fp16 probabilities


class Loop:
    """A pool with page tables on the device, and each sequence's tokens on the host."""

    def __init__(self, ops, dev, slots, seqs, width, seed):
        self.ops, self.dev = ops, dev
        self.gen = torch.Generator().manual_seed(seed)
        self.kv = torch.full((LAYERS, 2, slots, BLOCK, HEADS, DIM), float("nan"), dtype=torch.float16, device=dev)
        self.caches = ops.PlaneTable([self.kv[l, p] for p in range(2) for l in range(LAYERS)], 2)
        self.meta = torch.zeros(slots, dtype=torch.uint8, device=dev)
        self.l2p = torch.full((4 * slots,), -1, dtype=torch.int64, device=dev)
        self.p2l = torch.full((slots,), -1, dtype=torch.int64, device=dev)
        self.start = torch.zeros(1, dtype=torch.int64, device=dev)
        self.tables = torch.full((seqs, width), -1, dtype=torch.int64, device=dev)
        self.lens = torch.zeros(seqs, dtype=torch.int64, device=dev)
        self.next_id = 0
        self.text = [[] for _ in range(seqs)]  # per sequence: (K, V) of each token, (layers, heads, dim)

    def pool(self):
        return self.meta, self.l2p, self.p2l, self.tables, self.lens

    def ids(self, x):
        return torch.tensor(x, dtype=torch.int64, device=self.dev)

    def take(self, n):
        """n pinned slots, as the adapter's save takes them."""
        slots = self.ops.pop_reusable_slots(self.meta, self.start, self.ids([]), n)
        old = self.p2l[slots]
        new = torch.arange(self.next_id, self.next_id + n, device=self.dev)
        self.next_id += n
        ones = torch.ones(n, dtype=torch.uint8, device=self.dev)
        self.ops.commit_save_metadata(self.l2p, self.p2l, self.meta, old[old >= 0], new, slots, ones, ones)
        return slots

    def append(self, counts):
        """counts[s] new tokens of sequence s: pages, bytes, lengths."""
        mapping, rows = [], []
        for s, n in counts.items():
            have = len(self.text[s])
            need = -(-(have + n) // BLOCK) - -(-have // BLOCK)
            if need:
                first = -(-have // BLOCK)
                self.tables[s, first:first + need] = self.take(need)
            k = torch.randn((n, LAYERS, HEADS, DIM), generator=self.gen).half()
            v = torch.randn((n, LAYERS, HEADS, DIM), generator=self.gen).half()
            pos = torch.arange(have, have + n, device=self.dev)
            mapping.append(self.tables[s, pos // BLOCK] * BLOCK + pos % BLOCK)
            rows.append(torch.cat([k.transpose(0, 1), v.transpose(0, 1)]))  # (planes, n, heads, dim)
            self.text[s] = self.text[s] + [(k[i], v[i]) for i in range(n)]
            self.lens[s] = have + n
        self.ops.scatter_tokens(self.caches, torch.cat(mapping), torch.cat(rows, 1).unsqueeze(0).to(self.dev))

    def attend(self, counts, window=None, sinks=0):
        """Every layer's attention of the last counts[s] tokens, checked."""
        seqs = sorted(counts)
        new = [counts[s] for s in seqs]
        tables, lens = self.tables[self.ids(seqs)], self.lens[self.ids(seqs)]
        step = max(new) == 1
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        for layer in range(LAYERS):
            q = torch.randn((sum(new), HEADS * GROUP, DIM), generator=self.gen).half()
            args = (self.kv[layer, 0], self.kv[layer, 1], tables, lens)
            if step:
                out = self.ops.attend_step(q.to(self.dev), *args, window=window, sinks=sinks, check=True)
            else:
                out = self.ops.attend_chunk(q.to(self.dev), self.ids(offsets), *args, window=window, sinks=sinks,
                                            check=True)
            # the host's tokens as a cache of one-token blocks
            text = [t for s in seqs for t in self.text[s]]
            key = torch.stack([t[0][layer] for t in text]).unsqueeze(1)
            value = torch.stack([t[1][layer] for t in text]).unsqueeze(1)
            at, rows = 0, []
            for s in seqs:
                rows.append(torch.arange(at, at + len(self.text[s])))
                at += len(self.text[s])
            want, _, bound, _ = oracle.attention(q, key, value, rows, [len(self.text[s]) for s in seqs], new,
                                                 window=window, sinks=sinks, p_eps=P_EPS["step" if step else "chunk"])
            err = (out.cpu().double() - want).abs()
            assert torch.isfinite(err).all() and (err <= bound).all(), (err / bound).max()

    def check_pins(self):
        """Every slot is pinned by exactly the sequences that hold it."""
        want = torch.zeros(self.meta.numel(), dtype=torch.int64)
        for s, text in enumerate(self.text):
            for slot in self.tables[s, :-(-len(text) // BLOCK)].tolist():
                want[slot] += 1
        assert torch.equal((self.meta.cpu() & 15).long(), want)
        assert self.lens.tolist() == [len(t) for t in self.text]


def test_serving_loop():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    dev = torch.device("cuda", 0)
    loop = Loop(ops, dev, slots=120, seqs=9, width=12, seed=1)
    prompts = {0: 70, 1: 48, 2: 5}
    loop.append(prompts)
    loop.attend(prompts)
    loop.append({0: 30, 2: 41})  # the next piece of two prompts
    loop.attend({0: 30, 2: 41})
    loop.attend({0: 30, 2: 41}, window=25, sinks=3)
    loop.check_pins()
    # samples: 0 twice, 1 (whose last page is full) once, 2 once
    parents, children = [0, 1, 2, 0], [4, 5, 6, 7]
    fresh = ops.pop_reusable_slots(loop.meta, loop.start, loop.ids([]), 4)
    new_ids = loop.ids(range(loop.next_id, loop.next_id + 4))
    loop.next_id += 4
    ops.fork_sequences(*loop.pool(), loop.ids(parents), loop.ids(children), fresh, new_ids, loop.caches, check=True)
    for p, c in zip(parents, children):
        loop.text[c] = list(loop.text[p])
    loop.check_pins()
    live = [0, 1, 2, 4, 5, 6, 7]
    for _ in range(20):  # every sequence goes its own way, over page ends
        loop.append({s: 1 for s in live})
        loop.attend({s: 1 for s in live})
    loop.attend({s: 1 for s in live}, window=33, sinks=2)
    loop.check_pins()
    ops.free_sequences(*loop.pool(), loop.ids([0, 5, 2]), BLOCK, discard=True, check=True)
    for s in (0, 5, 2):
        loop.text[s] = []
    loop.check_pins()
    remap, count = ops.compact_pages(*loop.pool(), loop.caches, check=True)
    n = count.item()
    assert (loop.p2l[n:] == -1).all() and (loop.meta[n:] == 0).all()
    loop.check_pins()
    live = [1, 4, 6, 7]
    loop.attend({s: 1 for s in live})
    for _ in range(18):
        loop.append({s: 1 for s in live})
        loop.attend({s: 1 for s in live})
    # drafted tokens, verified in one chunk
    loop.append({1: 3, 4: 5, 6: 1, 7: 2})
    loop.attend({1: 3, 4: 5, 6: 1, 7: 2})
    loop.check_pins()


def test_calls_on_two_streams():
    """Steps and chunks in flight on two streams at once, and tensors used on a stream other than their own."""
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    dev = torch.device("cuda", 0)
    step = oracle.Batch(lens=[700, 33, 1200], heads=2, group=4, dim=128, block=16, dtype=torch.float16, seed=1)
    chunk = oracle.Batch(lens=[500, 260], new=[130, 260], heads=2, group=2, dim=64, block=16, dtype=torch.float16, seed=2)
    sk, sv = step.on(dev)
    ck, cv = chunk.on(dev)
    sq, cq = step.query.to(dev), chunk.query.to(dev)
    st, ct = step.tables.to(dev), chunk.tables.to(dev)
    sl, cl = torch.tensor(step.lens, device=dev), torch.tensor(chunk.lens, device=dev)
    offs = torch.tensor([0, 130, 390], device=dev)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((ops.attend_step(sq, sk, sv, st, sl, check=False),
                         ops.attend_chunk(cq, offs, ck, cv, ct, cl, check=False)))
    torch.cuda.synchronize()
    ops.check_status(dev)
    want, _, bound, _ = oracle.attention(step.query, step.key, step.value, step.tables.clamp(min=0), step.lens,
                                         [1, 1, 1], p_eps=P_EPS["step"])
    cwant, _, cbound, _ = oracle.attention(chunk.query, chunk.key, chunk.value, chunk.tables.clamp(min=0), chunk.lens,
                                           chunk.new, p_eps=P_EPS["chunk"])
    for s, c in outs:
        assert ((s.cpu().double() - want).abs() <= bound).all()
        assert ((c.cpu().double() - cwant).abs() <= cbound).all()


def test_pages_past_four_gigabytes():
    """Attention, a fork and a compaction over pages whose byte offsets need more than 32 bits."""
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    dev = torch.device("cuda", 0)
    slots = 1_100_000  # 4.5 GB per plane
    kv = torch.zeros((2, slots, 16, 1, 128), dtype=torch.float16, device=dev)
    pages = [slots - 1, 5, slots - 3, 1_060_000]
    g = torch.Generator(device=dev).manual_seed(4)
    for p in range(2):
        kv[p, pages] = torch.randn((4, 16, 1, 128), generator=g, device=dev).half()
    tables = torch.full((2, 4), -1, dtype=torch.int64, device=dev)
    tables[0] = torch.tensor(pages, device=dev)
    lens = torch.tensor([60, 0], device=dev)
    q = torch.randn((2, 2, 128), generator=g, device=dev).half()
    rows = kv[:, tables[0]].flatten(1, 2)[:, :60, 0].double()
    weight = torch.softmax(q[0].double() @ rows[0].T / 128 ** 0.5, -1)
    want, share = weight @ rows[1], weight @ rows[1].abs()
    bound = 2.0 ** -10 * share + 2.0 ** -11 * want.abs()  # probabilities and score sums, the result's rounding
    step = ops.attend_step(q, kv[0], kv[1], tables, lens, check=True)
    assert ((step[0].double() - want).abs() <= bound).all() and (step[1] == 0).all()
    chunk = ops.attend_chunk(q[:1].contiguous(), torch.tensor([0, 1, 1], device=dev), kv[0], kv[1], tables, lens,
                             check=True)
    assert ((chunk[0].double() - want).abs() <= bound).all()
    meta = torch.zeros(slots, dtype=torch.uint8, device=dev)
    l2p, p2l = (torch.full((n,), -1, dtype=torch.int64, device=dev) for n in (100, slots))
    held = torch.tensor(pages, device=dev)
    meta[held], p2l[held], l2p[:4] = 0x11, torch.arange(4, device=dev), held
    pool, one = (meta, l2p, p2l, tables, lens), torch.zeros(1, dtype=torch.int64, device=dev)
    ops.fork_sequences(*pool, one, one + 1, one + slots - 2, one + 50, [kv[0], kv[1]], check=True)
    both = ops.attend_step(q[:1].repeat(2, 1, 1), kv[0], kv[1], tables, lens, check=True)
    assert torch.equal(both[0], step[0]) and torch.equal(both[1], step[0])
    _, live = ops.compact_pages(*pool, [kv[0], kv[1]], check=True)
    assert live.item() == 5 and int(tables.max()) == 4
    both = ops.attend_step(q[:1].repeat(2, 1, 1), kv[0], kv[1], tables, lens, check=True)
    assert torch.equal(both[0], step[0]) and torch.equal(both[1], step[0])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_current():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    dev = torch.device("cuda", 1)
    torch.cuda.set_device(0)
    loop = Loop(ops, dev, slots=40, seqs=4, width=6, seed=3)
    loop.append({0: 40, 1: 7})
    loop.attend({0: 40, 1: 7})
    loop.append({0: 1, 1: 1})
    loop.attend({0: 1, 1: 1})
    ops.free_sequences(*loop.pool(), loop.ids([1]), BLOCK, discard=True, check=True)
    loop.text[1] = []
    ops.compact_pages(*loop.pool(), loop.caches, check=True)
    loop.attend({0: 1})
    assert torch.cuda.current_device() == 0
