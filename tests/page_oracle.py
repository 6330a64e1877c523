"""Sequences' pages in plain Python: the pool as lists, the operators by
their definitions, and a random pool to start from."""
from __future__ import annotations

import copy
import random

import torch


class Pool:
    def __init__(self, *, slots, logical, block, seqs, width, bits=8):
        self.slots, self.logical, self.block, self.bits = slots, logical, block, bits
        self.pin = [0] * slots
        self.usage = [0] * slots
        self.p2l = [-1] * slots
        self.l2p = [-1] * logical
        self.tables = [[-1] * width for _ in range(seqs)]
        self.lens = [0] * seqs

    def copy(self):
        return copy.deepcopy(self)

    def pages(self, s):
        return -(-max(self.lens[s], 0) // self.block)

    def fork(self, parents, children, fresh, ids, cache):
        """cache: (planes, slots, block, *row) tensor, changed in place."""
        for p, c, f, i in zip(parents, children, fresh, ids):
            full, rest = divmod(self.lens[p], self.block)
            for k in range(full):
                slot = self.tables[c][k] = self.tables[p][k]
                if slot >= 0:
                    self.pin[slot] += 1
            if rest:
                self.tables[c][full] = f
                if self.p2l[f] >= 0:
                    self.l2p[self.p2l[f]] = -1
                self.p2l[f], self.l2p[i] = i, f
                self.pin[f] = self.usage[f] = 1
                cache[:, f, :rest] = cache[:, self.tables[p][full], :rest]
            self.lens[c] = self.lens[p]

    def free(self, seqs, discard):
        for s in seqs:
            for k in range(self.pages(s)):
                slot, self.tables[s][k] = self.tables[s][k], -1
                if slot < 0:
                    continue
                self.pin[slot] -= 1
                if discard and self.pin[slot] == 0:
                    if self.p2l[slot] >= 0:
                        self.l2p[self.p2l[slot]] = -1
                    self.p2l[slot], self.usage[slot] = -1, 0
            if self.lens[s] > 0:
                self.lens[s] = 0

    def compact(self, cache):
        alive = [s for s in range(self.slots) if self.p2l[s] >= 0 or self.pin[s]]
        n = len(alive)
        remap = [-1] * self.slots
        for s in alive:
            remap[s] = s
        holes = [s for s in range(n) if remap[s] < 0]
        for d, s in zip(holes, [s for s in alive if s >= n]):
            remap[s] = d
            self.pin[d], self.usage[d], self.p2l[d] = self.pin[s], self.usage[s], self.p2l[s]
            self.pin[s] = self.usage[s] = 0
            self.p2l[s] = -1
            if self.p2l[d] >= 0:
                self.l2p[self.p2l[d]] = d
            cache[:, d] = cache[:, s]
        for s, row in enumerate(self.tables):
            for k in range(self.pages(s)):
                if row[k] >= 0:
                    row[k] = remap[row[k]]
        return remap, n

    def tensors(self, dev, stride=None):
        """slot_meta, l2p, p2l, block_tables, seq_lens on the device."""
        dtype = torch.uint8 if self.bits == 8 else torch.uint16
        meta = torch.tensor([p | u << (self.bits // 2) for p, u in zip(self.pin, self.usage)], dtype=torch.int32)
        tables = torch.tensor(self.tables).view(len(self.tables), -1)
        if stride:
            wide = torch.full((tables.shape[0], stride), 12345)
            wide[:, :tables.shape[1]] = tables
            tables = wide.to(dev)[:, :tables.shape[1]]
        return (meta.to(dtype).to(dev), torch.tensor(self.l2p, device=dev), torch.tensor(self.p2l, device=dev),
                tables.to(dev), torch.tensor(self.lens, device=dev))

    def assert_equal(self, tensors):
        meta, l2p, p2l, tables, lens = [t.cpu() for t in tensors]
        want = self.tensors("cpu")
        assert torch.equal(meta.to(torch.int32), want[0].to(torch.int32))
        assert torch.equal(l2p, want[1]) and torch.equal(p2l, want[2])
        assert torch.equal(tables, want[3].view_as(tables)) and torch.equal(lens, want[4])


def random_pool(seed, *, slots, seqs, longest, block, empty=3, bits=8, resident=0.3, shared=True, width_extra=2,
                gone=0.0):
    """`seqs` sequences with pages at random slots, some of them sharing a
    prefix, then `empty` empty ones; some unpinned resident blocks.  `gone`:
    share of the early pages that were given back."""
    r = random.Random(seed)
    lens = [r.randint(1, longest) for _ in range(seqs)]
    width = max([-(-n // block) for n in lens], default=0) + width_extra
    pool = Pool(slots=slots, logical=slots + 50, block=block, seqs=seqs + empty, width=width, bits=bits)
    free = list(range(slots))
    r.shuffle(free)
    ids = list(range(pool.logical))
    r.shuffle(ids)
    for s, n in enumerate(lens):
        common = []
        if shared and s % 3:
            lead = s - s % 3
            common = pool.tables[lead][:min(lens[lead], n) // block]
        for k in range(-(-n // block)):
            slot = common[k] if k < len(common) and common[k] >= 0 else free.pop()
            if r.random() < gone and k < n // block:
                if k >= len(common):
                    free.append(slot)
                slot = -1
            else:
                pool.pin[slot] += 1
            pool.tables[s][k] = slot
        pool.lens[s] = n
    for slot in range(slots):
        if pool.pin[slot] or (slot in free and r.random() < resident):
            pool.p2l[slot] = ids.pop()
            pool.l2p[pool.p2l[slot]] = slot
            pool.usage[slot] = r.randint(0, 7)
    pool.spare = free
    pool.unused_ids = ids
    return pool
