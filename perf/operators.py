"""Cases, plain forms and exact results of the paged-attention and page operators.

``attend_step`` (one new token per sequence over the paged cache),
``attend_chunk`` (a ragged chunk of new tokens per sequence),
``fork_sequences``, ``free_sequences`` and ``compact_pages``.  With ``own``
false, ``run`` computes each of them with elementary torch operations in 32
bits; with ``own`` true it makes the calls of ``kv_cache_adapter_cuda``.

Lengths follow from the case alone (``ragged`` seeds them); the values, the
order of the pages in the cache and the page tables follow from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "e4m3": torch.float8_e4m3fn}
PIN_MASK = 15


def listed():
    return [
        # A few chat turns on one Llama-3-70B KV-head shard (1 KV head, 8 query heads per GPU): the latency of one
        # decode step of one layer.
        dict(name="step-few", op="step", dtype="bfloat16", cache="bfloat16", seqs=4, heads=1, group=8, dim=128,
             block=16, min_len=90, max_len=900, window=0, sinks=0, idle=0, ragged=11),
        # An ordinary decode batch of the Llama-3-8B cache (8 KV heads, 32 query heads), ragged lengths, two slots of
        # the batch idle.
        dict(name="step-batch", op="step", dtype="float16", cache="float16", seqs=96, heads=8, group=4, dim=128,
             block=16, min_len=37, max_len=8191, window=0, sinks=0, idle=2, ragged=12),
        # Long contexts in an 8-bit cache of 64-token blocks, a sliding window with sinks for a large batch.
        dict(name="step-window-e4m3", op="step", dtype="bfloat16", cache="e4m3", seqs=256, heads=8, group=8, dim=128,
             block=64, min_len=500, max_len=16384, window=4096, sinks=4, idle=0, ragged=13),
        # Verification of a few drafted tokens per sequence: latency, few rows, split over the cache's length.
        dict(name="chunk-verify", op="chunk", dtype="float16", cache="float16", seqs=24, heads=8, group=4, dim=128,
             block=16, min_ctx=100, max_ctx=2500, min_new=1, max_new=8, window=0, sinks=0, ragged=21),
        # Prompts of the Llama-3-8B layout, one of them the continuation of a long prefix that the cache already holds.
        dict(name="chunk-prefill", op="chunk", dtype="bfloat16", cache="bfloat16", seqs=5, heads=8, group=4, dim=128,
             block=16, min_ctx=0, max_ctx=9000, min_new=700, max_new=4099, window=0, sinks=0, ragged=22),
        # Prompts through a sliding window with sinks, narrow heads, 8-bit cache.
        dict(name="chunk-window-e4m3", op="chunk", dtype="bfloat16", cache="e4m3", seqs=3, heads=4, group=6, dim=64,
             block=64, min_ctx=0, max_ctx=6000, min_new=1500, max_new=6001, window=1024, sinks=8, ragged=23),
        # Parallel sampling: a few prompts of the Llama-3-8B cache, every layer's last page copied per child.
        dict(name="fork-samples", op="fork", layers=32, heads=8, dim=128, block=16, slots=1024, parents=4, children=12,
             min_len=33, max_len=1500, ragged=31),
        # A beam step over a large batch of one-KV-head shards: mostly shared pages, many small copies.
        dict(name="fork-batch", op="fork", layers=32, heads=1, dim=128, block=16, slots=16384, parents=48, children=240,
             min_len=200, max_len=6000, ragged=32),
        # One finished request leaves; its pages stay resident for reuse.
        dict(name="free-one", op="free", slots=16384, block=16, seqs=24, freed=1, shared=0, discard=False,
             min_len=2000, max_len=9000, logical=20000, ragged=41),
        # Half of a large batch with long contexts and shared prefixes is dropped at once.
        dict(name="free-batch", op="free", slots=262144, block=16, seqs=256, freed=128, shared=3, discard=True,
             min_len=1000, max_len=32000, logical=400000, ragged=42),
        # A small pool after a burst: few pages move, every layer.
        dict(name="compact-small", op="compact", layers=32, heads=8, dim=128, block=16, slots=512, seqs=6, resident=20,
             min_len=20, max_len=500, ragged=51),
        # A large pool, a third of it live, before its tail is given back.
        dict(name="compact-large", op="compact", layers=32, heads=1, dim=128, block=16, slots=16384, seqs=64,
             resident=2500, min_len=50, max_len=2500, ragged=52),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["step", "step", "chunk", "chunk", "fork", "free", "compact"])
    ragged = rng.randrange(1 << 30)
    if op in ("step", "chunk"):
        dtype = rng.choice(["bfloat16", "float16"])
        cache = rng.choice([dtype, dtype, "e4m3"])
        dim = rng.choice([64, 80, 96, 112, 128, 128])
        block = rng.choice([1, 8, 16, 16, 32, 48, 64, 128])
        heads = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
        window, sinks = 0, 0
        if rng.random() < 0.4:
            window, sinks = _spread(rng, 1, 8000), rng.choice([0, 0, 1, 4, 17, 130])
        c = dict(op=op, dtype=dtype, cache=cache, heads=heads, group=group, dim=dim, block=block, window=window,
                 sinks=sinks, ragged=ragged)
        if op == "step":
            seqs = _spread(rng, 1, 256)
            longest = _spread(rng, 1, min(65536, 3_000_000 // (seqs * heads)))
            c.update(seqs=seqs, min_len=max(1, longest // rng.choice([1, 4, 30])), max_len=longest,
                     idle=rng.randrange(0, 3) if seqs > 3 else 0)
        else:
            seqs = _spread(rng, 1, 32)
            new = _spread(rng, 1, max(1, 8000 // seqs))
            # at most 1.2e9 (query head, key) pairs
            ctx = _spread(rng, 1, max(1, min(30000, 1_200_000_000 // (seqs * new * heads * group) - new)))
            c.update(seqs=seqs, min_ctx=rng.choice([0, 0, ctx // 2]), max_ctx=ctx, min_new=max(1, new // 3),
                     max_new=new)
        return c
    if op == "fork":
        heads, slots = rng.choice([(1, 8192), (2, 4096), (8, 1024)])
        parents = _spread(rng, 1, 16)
        longest = _spread(rng, 2, slots // 2 // parents * 16)
        return dict(op=op, layers=rng.choice([4, 17, 32]), heads=heads, dim=128, block=16, slots=slots,
                    parents=parents, children=rng.randrange(1, min(parents * 8, slots // 4) + 1),
                    min_len=max(1, longest // 5), max_len=longest, ragged=ragged)
    if op == "free":
        seqs = _spread(rng, 2, 256)
        longest = _spread(rng, 2, min(32000, 4_000_000 // seqs))
        block = rng.choice([1, 16, 16, 32, 64]) if longest <= 1000 else rng.choice([16, 32, 64])
        slots = seqs * (longest // block + 2) + rng.randrange(0, 5000)
        return dict(op=op, slots=slots, block=block, seqs=seqs, freed=rng.randrange(1, seqs + 1),
                    shared=rng.choice([0, 1, 3]), discard=rng.choice([True, False]), min_len=max(1, longest // 8),
                    max_len=longest, logical=slots + rng.randrange(1, 5000), ragged=ragged)
    heads, slots = rng.choice([(1, 8192), (2, 4096), (8, 1024)])
    seqs = _spread(rng, 1, 48)
    longest = _spread(rng, 2, slots // 2 // seqs * 16)
    return dict(op=op, layers=rng.choice([3, 16, 32]), heads=heads, dim=128, block=16, slots=slots, seqs=seqs,
                resident=rng.randrange(0, slots // 4), min_len=max(1, longest // 6), max_len=longest, ragged=ragged)


# ---------------------------------------------------------------------------
# lengths and work
# ---------------------------------------------------------------------------


def _lens(case):
    """(lengths, new tokens): the cached length of each sequence with the new tokens, and how many of them are new."""
    rng = random.Random(case["ragged"])
    op = case["op"]
    if op == "chunk":
        new = [_spread(rng, case["min_new"], case["max_new"]) for _ in range(case["seqs"])]
        ctx = [rng.randint(case["min_ctx"], case["max_ctx"]) for _ in range(case["seqs"])]
        return [c + n for c, n in zip(ctx, new)], new
    count = case["parents"] if op == "fork" else case["seqs"]
    lens = [_spread(rng, case["min_len"], case["max_len"]) for _ in range(count)]
    for i in range(case.get("idle", 0)):
        lens[1 + 2 * i if 1 + 2 * i < count else 0] = 0
    return lens, [1 if n else 0 for n in lens]


def _seen(p, window, sinks):
    """Tokens that a query at position p sees."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    op = case["op"]
    lens, new = _lens(case)
    if op in ("step", "chunk"):
        esz = 1 if case["cache"] == "e4m3" else 2
        hq = case["heads"] * case["group"]
        rows = sum(new)
        pairs = tokens = pages = 0
        for n, q in zip(lens, new):
            if not n:
                continue
            pairs += sum(_seen(p, case["window"], case["sinks"]) for p in range(n - q, n))
            first = max(0, n - q - case["window"] + 1) if case["window"] else 0
            seen = n - first + min(case["sinks"], first)
            tokens += seen
            pages += -(-seen // case["block"])
        kv = 2 * tokens * case["heads"] * case["dim"] * esz
        io = rows * hq * (2 * case["dim"] * 2 + 4)
        return {"bytes": kv + io + 8 * (pages + 2 * len(lens)), "flops": 4 * case["dim"] * hq * pairs}
    block = case["block"]
    pages = [-(-n // block) for n in lens]
    if op == "free":
        freed = _freed(case)
        n = sum(pages[i] for i in freed)
        return {"bytes": n * (8 + 8 + 2) + len(freed) * 24, "flops": n}
    row = case["heads"] * case["dim"] * 2 * case["layers"] * 2  # one token in every plane
    if op == "fork":
        parents = _parents(case)
        table = sum(pages[p] for p in parents)
        copied = sum(lens[p] % block for p in parents)
        return {"bytes": 16 * table + 2 * sum(pages[p] for p in set(parents)) + 2 * copied * row,
                "flops": table}
    live = sum(pages) + case["resident"]
    moved = live * (case["slots"] - live) // case["slots"]
    return {"bytes": 2 * moved * block * row + 9 * case["slots"] + 24 * moved + 16 * sum(pages),
            "flops": case["slots"]}


def _parents(case):
    got = [j % case["parents"] for j in range(case["children"])]
    random.Random(case["ragged"] + 1).shuffle(got)
    return got


def _freed(case):
    rng = random.Random(case["ragged"] + 1)
    return rng.sample(range(case["seqs"]), case["freed"])


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    st = _prepare_attention(case, gen, dev) if case["op"] in ("step", "chunk") else \
        _prepare_pages(case, seed, gen, dev)
    if own:
        from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

        st["ops"] = ops
        if "kv" in st:
            kv = st["kv"]
            st["caches"] = ops.PlaneTable([kv[l, p] for p in range(2) for l in range(kv.shape[0])], 2)
    return st


def _prepare_attention(case, gen, dev):
    lens, new = _lens(case)
    block, heads, group, dim = case["block"], case["heads"], case["group"], case["dim"]
    pages = [-(-n // block) for n in lens]
    spare = 1 + sum(pages) // 16
    slots = sum(pages) + spare
    order = torch.randperm(slots, generator=gen, device=dev)
    tables = torch.zeros((len(lens), max(1, max(pages))), dtype=torch.int64, device=dev)
    at = 0
    for i, n in enumerate(pages):
        tables[i, :n] = order[at:at + n]
        at += n
    dtype = DTYPES[case["dtype"]]

    def cache():
        t = torch.randn((slots, block, heads, dim), generator=gen, device=dev, dtype=torch.bfloat16)
        if case["cache"] != "e4m3":
            return t.to(DTYPES[case["cache"]])
        return (t * 16).to(DTYPES["e4m3"])

    key, value = cache(), cache()
    rows = len(lens) if case["op"] == "step" else sum(new)
    query = torch.randn((rows, heads * group, dim), generator=gen, device=dev).to(dtype)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    scale8 = 1.0 / 16 if case["cache"] == "e4m3" else 1.0
    return dict(case=case, query=query, key=key, value=value, tables=tables, lens_host=lens, new_host=new,
                lens=torch.tensor(lens, dtype=torch.int64, device=dev),
                offsets=torch.tensor(offsets, dtype=torch.int64, device=dev),
                out=torch.empty_like(query),
                lse=torch.empty(query.shape[:2], dtype=torch.float32, device=dev),
                key_scale=scale8, value_scale=scale8, scale=1.0 / math.sqrt(dim),
                window=case["window"] or None, sinks=case["sinks"])


def _prepare_pages(case, seed, gen, dev):
    """The pool's metadata in one buffer (``live``; ``start`` is what it holds before the call, copied back by each
    pass), the page tables, and the cache's planes where pages move."""
    op, block, slots = case["op"], case["block"], case["slots"]
    rng = random.Random(seed)
    lens, _ = _lens(case)
    pages = [-(-n // block) for n in lens]
    order = list(range(slots))
    rng.shuffle(order)
    take = iter(order)
    rows = case["parents"] + case["children"] if op == "fork" else case["seqs"]
    width = max(pages) + 3
    tables = torch.full((rows, width), -1, dtype=torch.int64)
    pins = [0] * slots
    prefix = {}
    for i, n in enumerate(pages):
        # with shared prefixes, each group of sequences starts with the full pages of its first member
        lead = i - i % (case.get("shared", 0) + 1)
        common = 0
        if lead != i:
            common = min(lens[i], lens[lead]) // block // 2
        got = prefix.get(lead, [])[:common] + [next(take) for _ in range(n - common)]
        if lead == i:
            prefix[i] = got
        tables[i, :n] = torch.tensor(got, dtype=torch.int64)
        for s in got:
            pins[s] += 1
    logical = case.get("logical", slots + 1000)
    ids = list(range(logical))
    rng.shuffle(ids)
    next_id = iter(ids)
    p2l = [-1] * slots
    usage = [0] * slots
    for s in range(slots):
        if pins[s]:
            p2l[s], usage[s] = next(next_id), 1 + s % 3
    resident = case.get("resident", slots // 16)
    spare = [s for s in take]
    for s in spare[:resident]:
        p2l[s], usage[s] = next(next_id), 1 + s % 5
    l2p = [-1] * logical
    for s, l in enumerate(p2l):
        if l >= 0:
            l2p[l] = s
    seq_lens = torch.zeros(rows, dtype=torch.int64)
    seq_lens[:len(lens)] = torch.tensor(lens, dtype=torch.int64)
    parts = dict(tables=tables, lens=seq_lens, l2p=torch.tensor(l2p), p2l=torch.tensor(p2l),
                 meta=torch.tensor([p | u << 4 for p, u in zip(pins, usage)], dtype=torch.uint8))
    start = torch.cat([t.contiguous().view(torch.uint8).flatten() for t in parts.values()]).to(dev)
    live = start.clone()
    st = dict(case=case, start=start, live=live)
    at = 0
    for name, t in parts.items():
        nbytes = t.numel() * t.element_size()
        st[name] = live[at:at + nbytes].view(t.dtype).view(t.shape)
        at += nbytes
    if op == "fork":
        parents = _parents(case)
        st["parents"] = torch.tensor(parents, device=dev)
        st["children"] = torch.tensor(rng.sample(range(case["parents"], rows), len(parents)), device=dev)
        # the pool hands out unpinned slots, some of which still hold an old logical block
        fresh = rng.sample(spare, len(parents))
        st["fresh"] = torch.tensor(fresh, device=dev)
        st["fresh_ids"] = torch.tensor([next(next_id) for _ in parents], device=dev)
        st["partial"] = torch.tensor([j for j, p in enumerate(parents) if lens[p] % block], dtype=torch.int64,
                                     device=dev)
    elif op == "free":
        st["freed"] = torch.tensor(_freed(case), device=dev)
    else:
        st["remap"] = torch.empty(slots, dtype=torch.int64, device=dev)
    if op != "free":
        st["kv"] = torch.empty((case["layers"], 2, slots, block, case["heads"], case["dim"]), dtype=torch.bfloat16,
                               device=dev).normal_(generator=gen)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if op in ("step", "chunk"):
        if own:
            return _own_attention(st)
        return _plain_step(st) if op == "step" else _plain_chunk(st)
    st["live"].copy_(st["start"])
    return (_own_pages if own else {"fork": _plain_fork, "free": _plain_free, "compact": _plain_compact}[op])(st)


def _own_attention(st):
    kw = dict(scale=st["scale"], window=st["window"], sinks=st["sinks"], key_scale=st["key_scale"],
              value_scale=st["value_scale"], out=st["out"], lse=st["lse"], check=False)
    if st["case"]["op"] == "step":
        st["ops"].attend_step(st["query"], st["key"], st["value"], st["tables"], st["lens"], **kw)
    else:
        st["ops"].attend_chunk(st["query"], st["offsets"], st["key"], st["value"], st["tables"], st["lens"], **kw)
    return st["out"], st["lse"]


def _own_pages(st):
    ops, op = st["ops"], st["case"]["op"]
    pool = (st["meta"], st["l2p"], st["p2l"], st["tables"], st["lens"])
    if op == "fork":
        ops.fork_sequences(*pool, st["parents"], st["children"], st["fresh"], st["fresh_ids"], st["caches"],
                           check=False)
        return (*pool, st["kv"])
    if op == "free":
        ops.free_sequences(*pool, st["freed"], st["case"]["block"], discard=st["case"]["discard"], check=False)
        return pool
    remap, live = ops.compact_pages(*pool, st["caches"], remap=st["remap"], check=False)
    return (*pool, remap, live, st["kv"])


def _plain_step(st):
    case, lens = st["case"], st["lens_host"]
    group, dev = case["group"], st["query"].device
    out = torch.zeros(st["query"].shape, dtype=torch.float32, device=dev)
    lse = torch.full(st["lse"].shape, -math.inf, dtype=torch.float32, device=dev)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        if case["window"] and n > case["window"]:
            pos = torch.cat([torch.arange(min(case["sinks"], n - case["window"]), device=dev),
                             torch.arange(n - case["window"], n, device=dev)])
        else:
            pos = torch.arange(n, device=dev)
        page, off = st["tables"][i][pos // case["block"]], pos % case["block"]
        k = st["key"][page, off].float() * st["key_scale"]  # (tokens, heads, dim)
        v = st["value"][page, off].float() * st["value_scale"]
        q = st["query"][i].float().view(case["heads"], group, case["dim"])
        s = torch.matmul(q, k.permute(1, 2, 0)) * st["scale"]
        m = s.amax(-1, keepdim=True)
        e = torch.exp(s - m)
        total = e.sum(-1, keepdim=True)
        out[i] = (torch.matmul(e, v.transpose(0, 1)) / total).view(-1, case["dim"])
        lse[i] = (m + torch.log(total)).view(-1)
    return out.to(st["query"].dtype), lse


def _plain_chunk(st):
    case, lens, new = st["case"], st["lens_host"], st["new_host"]
    group, dim, dev = case["group"], case["dim"], st["query"].device
    out = torch.zeros(st["query"].shape, dtype=torch.float32, device=dev)
    lse = torch.full(st["lse"].shape, -math.inf, dtype=torch.float32, device=dev)
    at = 0
    for i, (n, fresh) in enumerate(zip(lens, new)):
        pos = torch.arange(n, device=dev)
        page, off = st["tables"][i][pos // case["block"]], pos % case["block"]
        for h in range(case["heads"]):
            k = st["key"][page, off, h].float() * st["key_scale"]
            v = st["value"][page, off, h].float() * st["value_scale"]
            for a in range(0, fresh, 1024):
                b = min(a + 1024, fresh)
                p = torch.arange(n - fresh + a, n - fresh + b, device=dev).view(-1, 1)
                hidden = pos > p
                if case["window"]:
                    hidden |= (pos <= p - case["window"]) & (pos >= case["sinks"])
                rows = slice(at + a, at + b)
                heads = slice(h * group, (h + 1) * group)
                q = st["query"][rows, heads].float()
                s = torch.matmul(q.reshape(-1, dim), k.t()).view(b - a, group, n) * st["scale"]
                s = s.masked_fill(hidden.view(b - a, 1, n), -math.inf)
                m = s.amax(-1, keepdim=True)
                e = torch.exp(s - m)
                total = e.sum(-1, keepdim=True)
                out[rows, heads] = torch.matmul(e.view(-1, n), v).view(b - a, group, dim) / total
                lse[rows, heads] = (m + torch.log(total)).squeeze(-1)
        at += fresh
    return out.to(st["query"].dtype), lse


def _page_counts(tables, used, slots):
    """How often each slot stands at a marked place of the tables."""
    return torch.zeros(slots, dtype=torch.int64, device=tables.device).scatter_add_(
        0, tables.clamp(min=0).flatten(), used.long().flatten())


def _plain_fork(st):
    case, block = st["case"], st["case"]["block"]
    meta, l2p, p2l, tables, lens = st["meta"], st["l2p"], st["p2l"], st["tables"], st["lens"]
    n = lens[st["parents"]].view(-1, 1)
    rows = tables[st["parents"]]
    col = torch.arange(tables.shape[1], device=tables.device)
    counts = _page_counts(rows, col < n // block, case["slots"])
    meta.copy_((meta.long() + counts).to(torch.uint8))
    new_rows = torch.where(col < (n + block - 1) // block, rows, tables[st["children"]])
    part = st["partial"]
    fresh, ids = st["fresh"][part], st["fresh_ids"][part]
    last = n[part] // block
    source = rows[part].gather(1, last).view(-1)
    new_rows[part] = new_rows[part].scatter(1, last, fresh.view(-1, 1))
    tables[st["children"]] = new_rows
    lens[st["children"]] = n.view(-1)
    old = p2l[fresh]
    padded = torch.cat([l2p, l2p.new_zeros(1)])
    padded[torch.where(old >= 0, old, l2p.numel())] = -1
    padded[ids] = fresh
    l2p.copy_(padded[:-1])
    p2l[fresh] = ids
    meta[fresh] = 1 | 1 << 4
    filled = torch.arange(block, device=tables.device) < (n[part] % block)  # (copies, block)
    kv = st["kv"]
    for layer in range(kv.shape[0]):
        for plane in range(2):
            t = kv[layer, plane]
            t[fresh] = torch.where(filled.view(*filled.shape, 1, 1), t[source], t[fresh])
    return meta, l2p, p2l, tables, lens, kv


def _plain_free(st):
    case, block = st["case"], st["case"]["block"]
    meta, l2p, p2l, tables, lens = st["meta"], st["l2p"], st["p2l"], st["tables"], st["lens"]
    rows = tables[st["freed"]]
    n = lens[st["freed"]].view(-1, 1)
    used = torch.arange(tables.shape[1], device=tables.device) < (n + block - 1) // block
    counts = _page_counts(rows, used & (rows >= 0), case["slots"])
    left = meta.long() - counts
    gone = (counts > 0) & (left & PIN_MASK == 0)
    if case["discard"]:
        padded = torch.cat([l2p, l2p.new_zeros(1)])
        padded[torch.where(gone & (p2l >= 0), p2l, l2p.numel())] = -1
        l2p.copy_(padded[:-1])
        p2l.copy_(torch.where(gone, -1, p2l))
        left = torch.where(gone, 0, left)
    meta.copy_(left.to(torch.uint8))
    tables[st["freed"]] = torch.where(used, -1, rows)
    lens[st["freed"]] = 0
    return meta, l2p, p2l, tables, lens


def _plain_compact(st):
    case, block, slots = st["case"], st["case"]["block"], st["case"]["slots"]
    meta, l2p, p2l, tables, lens = st["meta"], st["l2p"], st["p2l"], st["tables"], st["lens"]
    index = torch.arange(slots, device=meta.device)
    live = (p2l >= 0) | (meta & PIN_MASK != 0)
    count = live.sum()
    src = torch.nonzero(live & (index >= count)).view(-1)
    dst = torch.nonzero(~live & (index < count)).view(-1)
    remap = torch.where(live, index, -1)
    remap[src] = dst
    used = torch.arange(tables.shape[1], device=meta.device) < (lens.view(-1, 1) + block - 1) // block
    tables.copy_(torch.where(used & (tables >= 0), remap[tables.clamp(min=0)], tables))
    ids = p2l[src]
    padded = torch.cat([l2p, l2p.new_zeros(1)])
    padded[torch.where(ids >= 0, ids, l2p.numel())] = dst
    l2p.copy_(padded[:-1])
    p2l[dst], meta[dst] = ids, meta[src]
    p2l[src], meta[src] = -1, 0
    kv = st["kv"]
    for layer in range(kv.shape[0]):
        for plane in range(2):
            kv[layer, plane][dst] = kv[layer, plane][src]
    return meta, l2p, p2l, tables, lens, remap, count.view(1), kv


# ---------------------------------------------------------------------------
# exact results
# ---------------------------------------------------------------------------


def exact(case, seed):
    """The operators by their definitions in 64 bits; moved cache bytes are not computed numbers (None)."""
    st = _prepare_attention(case, torch.Generator(device="cuda").manual_seed(seed), torch.device("cuda")) \
        if case["op"] in ("step", "chunk") else None
    if st is not None:
        return _exact_attention(st)
    dev = torch.device("cuda")
    st = _prepare_pages({**case, "layers": 1} if "layers" in case else case, seed,
                        torch.Generator(device="cuda").manual_seed(seed), dev)
    return {"fork": _exact_fork, "free": _exact_free, "compact": _exact_compact}[case["op"]](st)


def _exact_attention(st):
    case = st["case"]
    step = case["op"] == "step"
    window = case["window"] or 1 << 60
    out = torch.zeros(st["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["query"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, fresh) in enumerate(zip(st["lens_host"], st["new_host"])):
        row0 = i if step else first
        first += fresh
        if not n:
            continue
        low = max(0, n - fresh - window + 1)  # tokens before this are seen as sinks only
        j = torch.tensor([t for t in range(n) if t >= low or t < case["sinks"]], device="cuda")
        flat = st["tables"][i][j.div(case["block"], rounding_mode="floor")] * case["block"] + j.remainder(case["block"])
        k_all = st["key"].flatten(0, 1)[flat].double() * st["key_scale"]
        v_all = st["value"].flatten(0, 1)[flat].double() * st["value_scale"]
        for r0 in range(0, fresh, 512):
            r1 = min(fresh, r0 + 512)
            p = torch.arange(n - fresh + r0, n - fresh + r1, device="cuda")[:, None]
            seen = (j <= p) & ((p - j < window) | (j < case["sinks"]))
            for head in range(case["heads"] * case["group"]):
                kv_head = head // case["group"]
                q = st["query"][row0 + r0:row0 + r1, head].double()
                s = (q @ k_all[:, kv_head].T) * st["scale"]
                logs = torch.logsumexp(torch.where(seen, s, -math.inf), dim=1)
                weight = torch.where(seen, torch.exp(s - logs[:, None]), 0.0)
                out[row0 + r0:row0 + r1, head] = weight @ v_all[:, kv_head]
                lse[row0 + r0:row0 + r1, head] = logs
    return out, lse


def _host(st, *names):
    return [st[name].tolist() for name in names]


def _exact_pool(meta, l2p, p2l, tables, lens, *more):
    return (torch.tensor(meta, dtype=torch.uint8), torch.tensor(l2p), torch.tensor(p2l), torch.tensor(tables),
            torch.tensor(lens), *more)


def _exact_fork(st):
    block = st["case"]["block"]
    meta, l2p, p2l, tables, lens = _host(st, "meta", "l2p", "p2l", "tables", "lens")
    for p, c, f, new in zip(*_host(st, "parents", "children", "fresh", "fresh_ids")):
        for col in range(lens[p] // block):
            tables[c][col] = tables[p][col]
            meta[tables[p][col]] += 1
        if lens[p] % block:
            tables[c][lens[p] // block] = f
            if p2l[f] >= 0:
                l2p[p2l[f]] = -1
            p2l[f], l2p[new], meta[f] = new, f, 0x11
        lens[c] = lens[p]
    return _exact_pool(meta, l2p, p2l, tables, lens, None)


def _exact_free(st):
    block = st["case"]["block"]
    meta, l2p, p2l, tables, lens = _host(st, "meta", "l2p", "p2l", "tables", "lens")
    for q in st["freed"].tolist():
        for col in range(-(-lens[q] // block)):
            s = tables[q][col]
            tables[q][col] = -1
            if s < 0:
                continue
            meta[s] -= 1
            if meta[s] & PIN_MASK == 0 and st["case"]["discard"]:
                meta[s] = 0
                if p2l[s] >= 0:
                    l2p[p2l[s]] = -1
                p2l[s] = -1
        lens[q] = 0
    return _exact_pool(meta, l2p, p2l, tables, lens)


def _exact_compact(st):
    block = st["case"]["block"]
    meta, l2p, p2l, tables, lens = _host(st, "meta", "l2p", "p2l", "tables", "lens")
    alive = [s for s in range(len(p2l)) if p2l[s] >= 0 or meta[s] & PIN_MASK]
    count = len(alive)
    remap = [-1] * len(p2l)
    for s in alive:
        remap[s] = s
    here = set(alive)
    holes = [s for s in range(count) if s not in here]
    for d, s in zip(holes, [s for s in alive if s >= count]):
        remap[s] = d
        meta[d], meta[s] = meta[s], 0
        p2l[d], p2l[s] = p2l[s], -1
        if p2l[d] >= 0:
            l2p[p2l[d]] = d
    for row, n in zip(tables, lens):
        for col in range(-(-n // block)):
            if row[col] >= 0:
                row[col] = remap[row[col]]
    return _exact_pool(meta, l2p, p2l, tables, lens, torch.tensor(remap), torch.tensor([count]), None)
