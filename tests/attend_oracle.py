"""Plain 64-bit attention over a paged cache, with the error a result may have.

For each query the visible tokens are gathered one sequence at a time and the
softmax is computed in float64 on the CPU.  The bound counts the roundings of
the kernels: fp32 sums of the scores (head_dim terms, each at most 2^-23 of
the sum of magnitudes, truncated rather than rounded by the tensor cores),
the exponential (2^-22 and the rounding of its argument), one rounding of the
probabilities to ``p_eps`` (relative) and one of the result to its type.
"""
from __future__ import annotations

import math
import random

import torch


def attention(query, key_cache, value_cache, tables, lens, new, *, scale=None, window=None, sinks=0, key_scale=1.0,
              value_scale=1.0, p_eps):
    """query (rows, heads, dim) on the CPU: new[s] rows of sequence s in turn,
    the last of them at position lens[s] - 1.  Returns (out, lse, out bound,
    lse bound) in float64."""
    rows, heads, dim = query.shape
    block = key_cache.shape[1]
    group = heads // key_cache.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(query.shape, dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    eps = torch.finfo(query.dtype).eps
    tiny = 2.0 ** -24 if query.dtype == torch.float16 else 2.0 ** -126
    row = 0
    for s, (n, fresh) in enumerate(zip(lens, new)):
        for p in range(n - fresh, n):
            seen = [j for j in range(p + 1) if not window or j > p - window or j < sinks]
            if seen:
                j = torch.tensor(seen)
                page = tables[s][j // block]
                k = key_cache[page, j % block].double() * key_scale  # (tokens, kv heads, dim)
                v = value_cache[page, j % block].double() * value_scale
                k = k.repeat_interleave(group, dim=1).transpose(0, 1)  # (heads, tokens, dim)
                v = v.repeat_interleave(group, dim=1).transpose(0, 1)
                q = query[row].double()
                score = scale * (k @ q.unsqueeze(-1)).squeeze(-1)
                size = abs(scale) * (k.abs() @ q.abs().unsqueeze(-1)).squeeze(-1).amax(-1)
                lse[row] = torch.logsumexp(score, -1)
                w = torch.softmax(score, -1)
                out[row] = (w.unsqueeze(1) @ v).squeeze(1)
                spread = (dim + 4) * 2.0 ** -23 * size + 2.0 ** -22 * (2 + score.abs().amax(-1))
                lse_bound[row] = spread + 2.0 ** -22 * (1 + lse[row].abs()) + len(seen) * 2.0 ** -24
                share = (w.unsqueeze(1) @ v.abs()).squeeze(1)
                bound[row] = (share * (2 * spread + p_eps + len(seen) * 2.0 ** -23).unsqueeze(-1)
                              + eps / 2 * out[row].abs() * 1.01 + tiny)
            row += 1
    return out, lse, bound, lse_bound


class Batch:
    """A paged cache with the pages of some sequences at random places; every
    token that no query sees holds NaN or infinity, and so does every page no
    table names."""

    def __init__(self, *, lens, heads, group, dim, block, dtype, cache=None, new=None, window=None, sinks=0, seed=0,
                 layout="nhd", spare=3, extra_width=2, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.lens, self.new = lens, new if new is not None else [1 if n > 0 else 0 for n in lens]
        self.window, self.sinks = window, sinks
        e4m3 = cache == torch.float8_e4m3fn
        self.scales = dict(key_scale=0.0625, value_scale=0.25) if e4m3 else {}
        pages = [-(-max(n, 0) // block) for n in lens]
        slots = sum(pages) + spare
        order = torch.randperm(slots, generator=g)
        width = max(pages, default=0) + extra_width
        self.tables = torch.full((len(lens), width), -7, dtype=torch.int64)
        shape = (slots, block, heads, dim)
        poison = torch.tensor([math.nan, math.inf, -math.inf, math.nan])[torch.randint(0, 4, shape, generator=g)]
        if e4m3:
            poison = torch.full(shape, math.nan)
        k, v = poison.clone(), poison.flip(0).clone()
        at = 0
        for s, n in enumerate(lens):
            mine = order[at:at + pages[s]]
            at += pages[s]
            low = max(0, n - self.new[s] - window + 1) if window else 0
            for b in range(pages[s]):
                seen = [t for t in range(b * block, min(n, (b + 1) * block)) if t >= low or t < sinks]
                if not seen or self.new[s] == 0:
                    continue  # the page may have been given back: the entry stays invalid
                self.tables[s, b] = mine[b]
                off = torch.tensor(seen) % block
                scale = 16.0 if e4m3 else 1.0
                k[mine[b], off] = torch.randn((len(seen), heads, dim), generator=g) * scale * magnitude
                v[mine[b], off] = torch.randn((len(seen), heads, dim), generator=g) * scale
        self.key, self.value = k.to(cache), v.to(cache)
        rows = len(lens) if new is None else sum(self.new)
        self.query = torch.randn((rows, heads * group, dim), generator=g).to(dtype)
        self.layout = layout

    def on(self, dev):
        """(key, value) on the device in this batch's memory layout."""
        k, v = self.key, self.value
        if self.layout == "hnd":  # (blocks, heads, tokens, dim) in memory
            return (k.transpose(1, 2).contiguous().to(dev).transpose(1, 2),
                    v.transpose(1, 2).contiguous().to(dev).transpose(1, 2))
        if self.layout == "merged":  # one (blocks, tokens, 2, heads, dim) tensor
            both = torch.stack([k, v], 2).to(dev)
            return both[:, :, 0], both[:, :, 1]
        return k.to(dev), v.to(dev)

    def expect(self, p_eps, **kw):
        new = [1 if n > 0 else 0 for n in self.lens] if self.query.shape[0] == len(self.lens) else self.new
        rows = [s for s, n in enumerate(self.lens) if n > 0] if self.query.shape[0] == len(self.lens) else None
        q = self.query if rows is None else self.query[rows]
        return rows, attention(q, self.key, self.value, self.tables.clamp(min=0), self.lens, new, window=self.window,
                               sinks=self.sinks, p_eps=p_eps, **self.scales, **kw)


def random_lens(seed, count, longest):
    r = random.Random(seed)
    return [r.randint(1, longest) for _ in range(count)]
