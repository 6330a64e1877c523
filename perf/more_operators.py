"""Cases, plain forms and exact results of the token operators and of attention over 4-bit caches.

``rotate_tokens`` (rotary positions on rows of queries or keys, and their
transpose), ``append_tokens`` (rotated keys, values and queries of new tokens
into a paged cache of 16, 8 or 4 bits), ``read_tokens`` (rows of an 8- or 4-bit
cache as 16-bit values), and ``attend_step`` / ``attend_chunk`` over a cache
of 4 bits.  With ``own`` false, ``run`` computes each of them with elementary
torch operations in 32 bits; with ``own`` true it makes the calls of
``kv_cache_adapter_cuda``.

A 4-bit cache (``e2m1``) is uint8 ``(num_blocks, block_size, row)``: a token's
row holds the e2m1 codes of all heads (two per byte, the first in the low half),
then an e4m3 scale for each 16 values, and zeros up to a multiple of 16 bytes.

Lengths follow from the case alone (``ragged`` seeds them); the values, the
order of the pages in the cache and the page tables follow from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32,
          "e4m3": torch.float8_e4m3fn}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
TABLE = 32768  # positions in the rotation's table


def listed():
    return [
        # One decode step of a few chat turns on one Llama-3-70B KV-head shard: rotate the new tokens' queries and keys
        # and store keys and values; latency.
        dict(name="append-few", op="append", dtype="bfloat16", cache="bfloat16", rows=4, heads=1, group=8, dim=128,
             block=16, rotary=128, interleaved=False, pad=0, seqs=4, ragged=11),
        # Prompts of the Llama-3-8B layout (8 KV heads, 32 query heads), queries and keys as they lie in the output of
        # one projection.
        dict(name="append-prompt", op="append", dtype="bfloat16", cache="bfloat16", rows=16384, heads=8, group=4,
             dim=128, block=16, rotary=128, interleaved=False, pad=0, seqs=5, ragged=12),
        # A padded batch into an 8-bit cache of 64-token blocks, neighbouring dims rotated, half of the head only.
        dict(name="append-e4m3", op="append", dtype="float16", cache="e4m3", rows=2047, heads=4, group=6, dim=128,
             block=64, rotary=64, interleaved=True, pad=3, seqs=40, ragged=13),
        # Prompts into a 4-bit cache, and the stored rows read back.
        dict(name="append-e2m1", op="append", dtype="bfloat16", cache="e2m1", rows=8191, heads=8, group=4, dim=128,
             block=16, rotary=128, interleaved=False, pad=1, seqs=9, ragged=14),
        # Queries of a few drafted tokens by themselves.
        dict(name="rotate-few", op="rotate", dtype="float16", rows=48, heads=32, dim=128, rotary=128,
             interleaved=False, transpose=False, ragged=21),
        # The gradient of a long prompt's rotated queries.
        dict(name="rotate-gradient", op="rotate", dtype="float32", rows=8192, heads=32, dim=128, rotary=96,
             interleaved=True, transpose=True, ragged=22),
        # A short sequence leaves an 8-bit cache.
        dict(name="read-e4m3", op="read", dtype="float16", cache="e4m3", rows=700, heads=8, dim=128, block=16,
             ragged=31),
        # Long prefixes of a 4-bit cache, widened for another kernel or another cache.
        dict(name="read-e2m1", op="read", dtype="bfloat16", cache="e2m1", rows=65536, heads=8, dim=128, block=16,
             ragged=32),
        # Decode over a 4-bit cache: the latency of a few chat turns on one KV head.
        dict(name="step-few-e2m1", op="step", dtype="bfloat16", heads=1, group=8, dim=128, block=16, seqs=4,
             min_len=90, max_len=900, window=0, sinks=0, idle=0, ragged=41),
        # A large decode batch with long contexts, a sliding window with sinks.
        dict(name="step-window-e2m1", op="step", dtype="bfloat16", heads=8, group=8, dim=128, block=64, seqs=256,
             min_len=500, max_len=16384, window=4096, sinks=4, idle=2, ragged=42),
        # Verification of a few drafted tokens per sequence.
        dict(name="chunk-verify-e2m1", op="chunk", dtype="float16", heads=8, group=4, dim=128, block=16, seqs=24,
             min_ctx=100, max_ctx=2500, min_new=1, max_new=8, window=0, sinks=0, ragged=51),
        # Prompts, one of them the continuation of a long prefix that the cache already holds.
        dict(name="chunk-prefill-e2m1", op="chunk", dtype="bfloat16", heads=8, group=4, dim=128, block=16, seqs=4,
             min_ctx=0, max_ctx=7000, min_new=500, max_new=3001, window=0, sinks=0, ragged=52),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "append", "append", "rotate", "read", "step", "step", "chunk"])
    ragged = rng.randrange(1 << 30)
    dtype = rng.choice(["bfloat16", "float16"])
    block = rng.choice([1, 8, 16, 16, 32, 48, 64, 128])
    if op in ("append", "rotate"):
        cache = rng.choice([dtype, "e4m3", "e2m1"]) if op == "append" else None
        dim = rng.choice([32, 64, 96, 128, 128, 256]) if cache == "e2m1" else rng.choice([64, 80, 96, 112, 128, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
        heads = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
        c = dict(op=op, dtype=dtype, dim=dim, rotary=rotary, interleaved=rng.random() < 0.4, ragged=ragged)
        if op == "rotate":
            heads *= group
            c.update(dtype=rng.choice([dtype, dtype, "float32"]), rows=_spread(rng, 1, 30_000_000 // (heads * dim)),
                     heads=heads, transpose=rng.random() < 0.4)
        else:
            rows = _spread(rng, 1, min(16384, 80_000_000 // (heads * (group + 2) * dim)))
            c.update(cache=cache, rows=rows, heads=heads, group=group, block=block, pad=rng.choice([0, 0, 1, 4]),
                     seqs=_spread(rng, 1, min(rows, 64)))
        return c
    if op == "read":
        cache = rng.choice(["e4m3", "e2m1"])
        dim = rng.choice([32, 64, 96, 128, 128, 256]) if cache == "e2m1" else rng.choice([64, 80, 96, 112, 128, 128, 256])
        heads = rng.choice([1, 2, 3, 4, 8])
        return dict(op=op, dtype=rng.choice(["bfloat16", "float16", "float32"]), cache=cache, dim=dim, heads=heads,
                    block=block, rows=_spread(rng, 1, min(65536, 50_000_000 // (heads * dim))), ragged=ragged)
    heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    window, sinks = 0, 0
    if rng.random() < 0.4:
        window, sinks = _spread(rng, 1, 8000), rng.choice([0, 0, 1, 4, 17, 130])
    c = dict(op=op, dtype=dtype, heads=heads, group=group, block=block, window=window, sinks=sinks, ragged=ragged)
    if op == "step":
        seqs = _spread(rng, 1, 256)
        longest = _spread(rng, 1, min(65536, 3_000_000 // (seqs * heads)))
        c.update(dim=rng.choice([32, 64, 96, 128, 128, 256]), seqs=seqs,
                 min_len=max(1, longest // rng.choice([1, 4, 30])), max_len=longest,
                 idle=rng.randrange(0, 3) if seqs > 3 else 0)
    else:
        seqs = _spread(rng, 1, 32)
        new = _spread(rng, 1, max(1, 6000 // seqs))
        # at most 0.5e9 (query head, key) pairs
        ctx = _spread(rng, 1, max(1, min(30000, 500_000_000 // (seqs * new * heads * group) - new)))
        c.update(dim=rng.choice([32, 64, 96, 128, 128]), seqs=seqs, min_ctx=rng.choice([0, 0, ctx // 2]), max_ctx=ctx,
                 min_new=max(1, new // 3), max_new=new)
    return c


# ---------------------------------------------------------------------------
# lengths and work
# ---------------------------------------------------------------------------


def _row_bytes(heads, dim):
    return -(-heads * dim * 9 // 16 // 16) * 16


def _held(case, dtype):
    """Bytes of one token's keys (or values) in the cache."""
    values = case["heads"] * case["dim"]
    return {"e4m3": values, "e2m1": values * 9 // 16, "float32": 4 * values}.get(dtype, 2 * values)


def _lens(case):
    """(lengths, new tokens): the cached length of each sequence with the new tokens, and how many of them are new."""
    rng = random.Random(case["ragged"])
    if case["op"] == "chunk":
        new = [_spread(rng, case["min_new"], case["max_new"]) for _ in range(case["seqs"])]
        ctx = [rng.randint(case["min_ctx"], case["max_ctx"]) for _ in range(case["seqs"])]
        return [c + n for c, n in zip(ctx, new)], new
    lens = [_spread(rng, case["min_len"], case["max_len"]) for _ in range(case["seqs"])]
    for i in range(case.get("idle", 0)):
        lens[1 + 2 * i if 1 + 2 * i < len(lens) else 0] = 0
    return lens, [1 if n else 0 for n in lens]


def _positions(case):
    """The position of each new token: sequences of even shares of the rows, each after a context of its own."""
    rng = random.Random(case["ragged"])
    seqs = case.get("seqs", max(1, min(8, case["rows"] // 100)))
    got = []
    for s in range(seqs):
        count = case["rows"] * (s + 1) // seqs - case["rows"] * s // seqs
        first = rng.randint(0, TABLE - count)
        got += range(first, first + count)
    return got


def _seen(p, window, sinks):
    """Tokens that a query at position p sees."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    op, dim = case["op"], case["dim"]
    wide = 4 if case["dtype"] == "float32" else 2
    if op == "rotate":
        x = case["rows"] * case["heads"]
        return {"bytes": 2 * x * dim * wide + case["rows"] * (8 + 4 * case["rotary"]), "flops": 3 * x * case["rotary"]}
    if op == "append":
        rows = case["rows"] - len(_padding(case))
        q, kv = rows * case["heads"] * case["group"] * dim, 2 * rows * case["heads"] * dim
        held = 2 * rows * _held(case, case["cache"])
        back = held + 2 * kv if case["cache"] == "e2m1" else 0  # the stored rows read
        return {"bytes": 4 * q + 2 * kv + held + back + rows * 4 * case["rotary"] + 16 * case["rows"],
                "flops": 3 * (q + kv // 2) * case["rotary"] // dim}
    if op == "read":
        values = case["rows"] * case["heads"] * dim
        return {"bytes": case["rows"] * (8 + _held(case, case["cache"])) + wide * values, "flops": values}
    lens, new = _lens(case)
    hq = case["heads"] * case["group"]
    pairs = tokens = pages = 0
    for n, q in zip(lens, new):
        if not n:
            continue
        pairs += sum(_seen(p, case["window"], case["sinks"]) for p in range(n - q, n))
        first = max(0, n - q - case["window"] + 1) if case["window"] else 0
        seen = n - first + min(case["sinks"], first)
        tokens += seen
        pages += -(-seen // case["block"])
    kv = 2 * tokens * _held(case, "e2m1")
    return {"bytes": kv + sum(new) * hq * (4 * dim + 4) + 8 * (pages + 2 * len(lens)), "flops": 4 * dim * hq * pairs}


def _padding(case):
    """Rows of a padded batch that stand for no token."""
    return random.Random(case["ragged"] + 1).sample(range(case["rows"]), case["rows"] * case["pad"] // 16)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    return {"rotate": _prepare_rotate, "append": _prepare_append, "read": _prepare_read}.get(
        case["op"], _prepare_attention)(case, gen, dev)


def _angles(rotary, dev):
    """Cosines, then sines, of every position (base 500,000)."""
    rate = 500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=dev) / rotary)
    angle = torch.arange(TABLE, dtype=torch.float64, device=dev)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _cache(kind, slots, block, heads, dim, gen, dev):
    """A paged cache that holds tokens already (normal values; 8 bits: times 16)."""
    if kind != "e2m1":
        t = torch.randn((slots, block, heads, dim), generator=gen, device=dev, dtype=torch.bfloat16)
        return t.to(DTYPES[kind]) if kind != "e4m3" else (t * 16).to(DTYPES[kind])
    rows = torch.zeros((slots, block, _row_bytes(heads, dim)), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 26) // (block * heads * dim))
    for a in range(0, slots, step):
        part = rows[a:a + step]
        x = torch.randn((part.shape[0] * block, heads, dim), generator=gen, device=dev)
        part.view(-1, part.shape[2])[:, :heads * dim * 9 // 16] = _to_e2m1(x, 1.0)
    return rows


def _prepare_rotate(case, gen, dev):
    shape = (case["rows"], case["heads"], case["dim"])
    x = torch.randn(shape, generator=gen, device=dev).to(DTYPES[case["dtype"]])
    return dict(case=case, x=x, table=_angles(case["rotary"], dev), out=torch.empty_like(x),
                positions=torch.tensor(_positions(case), dtype=torch.int64, device=dev))


def _prepare_append(case, gen, dev):
    rows, heads, group, dim = case["rows"], case["heads"], case["group"], case["dim"]
    both = torch.randn((rows, (group + 2) * heads, dim), generator=gen, device=dev).to(DTYPES[case["dtype"]])
    slots = -(-rows // case["block"]) + 3
    key, value = (_cache(case["cache"], slots, case["block"], heads, dim, gen, dev) for _ in range(2))
    # pages in any order, filled one after the other
    order = torch.randperm(slots, generator=gen, device=dev)
    t = torch.arange(rows, device=dev)
    mapping = order[t // case["block"]] * case["block"] + t % case["block"]
    padding = torch.tensor(_padding(case), dtype=torch.int64, device=dev)
    mapping[padding] = -1
    return dict(case=case, query=both[:, :heads * group], key=both[:, heads * group:heads * (group + 1)],
                value=both[:, heads * (group + 1):], key_cache=key, value_cache=value, mapping=mapping,
                live=torch.nonzero(mapping >= 0).view(-1), table=_angles(case["rotary"], dev),
                positions=torch.tensor(_positions(case), dtype=torch.int64, device=dev),
                query_out=torch.zeros((rows, heads * group, dim), dtype=both.dtype, device=dev),
                factor=1.0 / 16 if case["cache"] == "e4m3" else 1.0,
                back=[torch.zeros((rows, heads, dim), dtype=both.dtype, device=dev) for _ in range(2)])


def _prepare_read(case, gen, dev):
    rows, block = case["rows"], case["block"]
    slots = -(-rows // block) + 3
    cache = _cache(case["cache"], slots, block, case["heads"], case["dim"], gen, dev)
    order = torch.randperm(slots, generator=gen, device=dev)
    t = torch.arange(rows, device=dev)
    return dict(case=case, cache=cache, mapping=order[t // block] * block + t % block,
                factor=1.0 / 16 if case["cache"] == "e4m3" else 1.0,
                out=torch.empty((rows, case["heads"], case["dim"]), dtype=DTYPES[case["dtype"]], device=dev))


def _prepare_attention(case, gen, dev):
    lens, new = _lens(case)
    block, heads, group, dim = case["block"], case["heads"], case["group"], case["dim"]
    pages = [-(-n // block) for n in lens]
    slots = sum(pages) + 1 + sum(pages) // 16
    order = torch.randperm(slots, generator=gen, device=dev)
    width = max(1, max(pages))
    counts = torch.tensor(pages, device=dev)
    col = torch.arange(width, device=dev)
    tables = torch.where(col < counts[:, None], order[((counts.cumsum(0) - counts)[:, None] + col).clamp(max=slots - 1)],
                         0)
    key, value = (_cache("e2m1", slots, block, heads, dim, gen, dev) for _ in range(2))
    rows = len(lens) if case["op"] == "step" else sum(new)
    query = torch.randn((rows, heads * group, dim), generator=gen, device=dev).to(DTYPES[case["dtype"]])
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    return dict(case=case, query=query, key=key, value=value, tables=tables, lens_host=lens, new_host=new,
                lens=torch.tensor(lens, dtype=torch.int64, device=dev),
                offsets=torch.tensor(offsets, dtype=torch.int64, device=dev), out=torch.empty_like(query),
                lse=torch.empty(query.shape[:2], dtype=torch.float32, device=dev), scale=1.0 / math.sqrt(dim),
                window=case["window"] or None, sinks=case["sinks"])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if own:
        return {"rotate": _own_rotate, "append": _own_append, "read": _own_read, "step": _own_step,
                "chunk": _own_chunk}[op](st)
    return {"rotate": _plain_rotate, "append": _plain_append, "read": _plain_read, "step": _plain_step,
            "chunk": _plain_chunk}[op](st)


def _ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


def _own_rotate(st):
    case = st["case"]
    return _ops().rotate_tokens(st["x"], st["positions"], st["table"], interleaved=case["interleaved"],
                                transpose=case["transpose"], out=st["out"], check=False)


def _own_append(st):
    ops, case = _ops(), st["case"]
    ops.append_tokens(st["key"], st["value"], st["key_cache"], st["value_cache"], st["mapping"],
                      positions=st["positions"], table=st["table"], interleaved=case["interleaved"],
                      query=st["query"], query_out=st["query_out"], key_scale=st["factor"], value_scale=st["factor"],
                      check=False)
    if case["cache"] != "e2m1":
        return st["query_out"], st["key_cache"], st["value_cache"]
    for cache, out in zip((st["key_cache"], st["value_cache"]), st["back"]):
        ops.read_tokens(cache, st["mapping"], head_dim=case["dim"], out=out, check=False)
    return st["query_out"], *st["back"]


def _own_read(st):
    return _ops().read_tokens(st["cache"], st["mapping"], head_dim=st["case"]["dim"], scale=st["factor"],
                              out=st["out"], check=False)


def _own_step(st):
    _ops().attend_step(st["query"], st["key"], st["value"], st["tables"], st["lens"], scale=st["scale"],
                       window=st["window"], sinks=st["sinks"], out=st["out"], lse=st["lse"], check=False)
    return st["out"], st["lse"]


def _own_chunk(st):
    _ops().attend_chunk(st["query"], st["offsets"], st["key"], st["value"], st["tables"], st["lens"],
                        scale=st["scale"], window=st["window"], sinks=st["sinks"], out=st["out"], lse=st["lse"],
                        check=False)
    return st["out"], st["lse"]


def _rotated(x, positions, table, interleaved, transpose):
    """x (rows, heads, dim) in 32 bits, its first dims rotated by the table's angles."""
    x = x.float()
    n = table.shape[1] // 2
    angle = table[positions][:, None]
    c, s = angle[..., :n], angle[..., n:]
    if transpose:
        s = -s
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    y, z = a * c - b * s, b * c + a * s
    turned = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _to_e2m1(x, factor):
    """Codes and scales of rows x (rows, heads, dim): bytes of (rows, heads * dim * 9 / 16)."""
    g = x.unflatten(-1, (-1, 16))
    six = torch.full((), 6 * factor, device=x.device)  # (a quotient by a number of the host is a product in torch)
    scale = (g.abs().amax(-1) / six).clamp(max=448).to(torch.float8_e4m3fn)
    unit = (scale.float() * factor)[..., None]
    y = torch.where(unit > 0, g / unit, 0.0)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + torch.signbit(y).byte() * 8)
    code = code.view(x.shape[0], -1)
    return torch.cat([code[:, 0::2] | code[:, 1::2] << 4, scale.view(torch.uint8).view(x.shape[0], -1)], 1)


def _from_e2m1(rows, heads, dim):
    """The values (..., heads, dim) of rows of bytes, in 32 bits."""
    n = heads * dim // 2
    codes = rows[..., :n]
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    values = torch.tensor(E2M1 + [-v for v in E2M1], device=rows.device)[codes]
    scale = rows[..., n:n + heads * dim // 16].contiguous().view(torch.float8_e4m3fn).float()
    return (values.unflatten(-1, (-1, 16)) * scale[..., None]).view(*rows.shape[:-1], heads, dim)


def _plain_rotate(st):
    case = st["case"]
    return _rotated(st["x"], st["positions"], st["table"], case["interleaved"], case["transpose"]).to(st["x"].dtype)


def _plain_append(st):
    case, live = st["case"], st["live"]
    at, turn = st["mapping"][live], (st["positions"][live], st["table"], case["interleaved"], False)
    st["query_out"][live] = _rotated(st["query"][live], *turn).to(st["query"].dtype)
    for cache, x in ((st["key_cache"], _rotated(st["key"][live], *turn)), (st["value_cache"], st["value"][live].float())):
        if case["cache"] == "e2m1":
            cache.view(-1, cache.shape[2])[at, :case["heads"] * case["dim"] * 9 // 16] = _to_e2m1(x, 1.0)
        elif case["cache"] == "e4m3":
            x8 = (x / torch.full((), st["factor"], device=x.device)).clamp(-448, 448).to(torch.float8_e4m3fn)
            cache.view(torch.uint8).flatten(0, 1)[at] = x8.view(torch.uint8)
        else:
            cache.flatten(0, 1)[at] = x.to(cache.dtype)
    if case["cache"] != "e2m1":
        return st["query_out"], st["key_cache"], st["value_cache"]
    for cache, out in zip((st["key_cache"], st["value_cache"]), st["back"]):
        out[live] = _from_e2m1(cache.view(-1, cache.shape[2])[at], case["heads"], case["dim"]).to(out.dtype)
    return st["query_out"], *st["back"]


def _plain_read(st):
    case, at = st["case"], st["mapping"]
    if case["cache"] == "e2m1":
        x = _from_e2m1(st["cache"].view(-1, st["cache"].shape[2])[at], case["heads"], case["dim"])
    else:
        x = st["cache"].view(torch.uint8).flatten(0, 1)[at].view(torch.float8_e4m3fn).float() * st["factor"]
    return x.to(st["out"].dtype)


def _plain_step(st):
    case, tables, lens = st["case"], st["tables"], st["lens"]
    heads, group, dim, block, window, sinks = (case[n] for n in ("heads", "group", "dim", "block", "window", "sinks"))
    longest = tables.shape[1] * block
    col = torch.arange(min(longest, window + sinks) if window else longest, device=lens.device)
    # the tokens that each sequence's last one sees, in front; the rest hidden
    gap = (lens - window - sinks).clamp(min=0)[:, None] if window else torch.zeros_like(lens)[:, None]
    pos = torch.where(col < sinks, col, col + gap) if window else col.expand(lens.shape[0], -1)
    hidden = pos >= lens[:, None]
    pos = torch.where(hidden, 0, pos)
    page = tables.gather(1, pos // block)
    k = _from_e2m1(st["key"][page, pos % block], heads, dim)  # (seqs, tokens, heads, dim)
    q = st["query"].float().view(-1, heads, group, dim)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * st["scale"]
    del k
    s = s.masked_fill(hidden[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    v = _from_e2m1(st["value"][page, pos % block], heads, dim)
    out = torch.matmul(e, v.transpose(1, 2)) / torch.where(total > 0, total, 1.0)
    return out.view(st["query"].shape).to(st["query"].dtype), (m + torch.log(total)).view(st["lse"].shape)


def _plain_chunk(st):
    case = st["case"]
    heads, group, dim, block, window, sinks = (case[n] for n in ("heads", "group", "dim", "block", "window", "sinks"))
    dev = st["query"].device
    outs, logs, at = [], [], 0
    for i, (n, fresh) in enumerate(zip(st["lens_host"], st["new_host"])):
        pos = torch.arange(n, device=dev)
        page = st["tables"][i][pos // block]
        k, v = (_from_e2m1(c[page, pos % block], heads, dim).transpose(0, 1) for c in (st["key"], st["value"]))
        p = pos[n - fresh:, None]
        hidden = pos > p
        if window:
            hidden |= (pos <= p - window) & (pos >= sinks)
        q = st["query"][at:at + fresh].float().view(fresh, heads, group * dim).transpose(0, 1)
        s = torch.matmul(q.reshape(heads, fresh * group, dim), k.transpose(1, 2)) * st["scale"]
        s = s.view(heads, fresh, group, n).masked_fill_(hidden[:, None], -math.inf)
        m = s.amax(-1, keepdim=True)
        e = torch.exp(s - m)
        total = e.sum(-1, keepdim=True)
        o = torch.matmul(e.view(heads, fresh * group, n), v).view(heads, fresh, group, dim) / total
        outs.append(o.transpose(0, 1).reshape(fresh, heads * group, dim))
        logs.append((m + torch.log(total)).transpose(0, 1).reshape(fresh, heads * group))
        at += fresh
    return torch.cat(outs).to(st["query"].dtype), torch.cat(logs)


# ---------------------------------------------------------------------------
# exact results
# ---------------------------------------------------------------------------


def exact(case, seed):
    """The operators by their definitions in 64 bits."""
    dev = torch.device("cuda")
    st = prepare(case, seed)
    if case["op"] == "rotate":
        return _turn64(st["x"], st, case["transpose"])
    if case["op"] == "append":
        return _exact_append(st)
    if case["op"] == "read":
        rows = st["cache"].flatten(0, 1)[st["mapping"]] if case["cache"] == "e2m1" else None
        if rows is None:
            return st["cache"].double().flatten(0, 1)[st["mapping"]] * st["factor"]
        return _values64(rows, case["heads"], case["dim"])
    return _exact_attention(st, dev)


def _turn64(x, st, transpose):
    """One pair of dims at a time as a complex number times exp(i angle) (its conjugate if transposed)."""
    case, x = st["case"], x.double().clone()
    n = case["rotary"] // 2
    turn = st["table"].double()[st["positions"]]
    turn = torch.complex(turn[:, :n], -turn[:, n:] if transpose else turn[:, n:])
    for i in range(n):
        d, e = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + n)
        z = torch.complex(x[:, :, d], x[:, :, e]) * turn[:, i:i + 1]
        x[:, :, d], x[:, :, e] = z.real, z.imag
    return x


def _grid64(x, bits, least):
    """x rounded to the nearest value of `bits` significant bits, the exponent at least `least`; ties to even."""
    e = torch.frexp(x.abs().clamp(min=1e-300)).exponent.long() - 1
    step = torch.exp2((e.clamp(min=least) - (bits - 1)).double())
    return torch.round(x / step) * step


def _stored64(x, kind, factor):
    """What a cache of `kind` gives back for x, in units of the factor for e4m3."""
    if kind == "e4m3":
        return _grid64(x / factor, 4, -6).clamp(-448, 448)
    if kind != "e2m1":
        return x
    g = x.unflatten(-1, (-1, 16))
    unit = _grid64(g.abs().amax(-1, keepdim=True) / 6, 4, -6).clamp(max=448)
    return (_grid64(g / unit.clamp(min=1e-300), 2, 0).clamp(-6, 6) * unit).flatten(-2)


def _exact_append(st):
    case, live = st["case"], st["live"]
    rows = [_turn64(st["query"], st, False), _turn64(st["key"], st, False), st["value"].double()]
    out = st["query_out"].double()
    out[live] = rows[0][live]
    got = [out]
    for cache, back, x in zip((st["key_cache"], st["value_cache"]), st["back"], rows[1:]):
        held = _stored64(x, case["cache"], st["factor"])
        to = back.double() if case["cache"] == "e2m1" else cache.double()
        if case["cache"] == "e2m1":
            to[live] = held[live]
        else:
            to.view(-1, case["heads"], case["dim"])[st["mapping"][live]] = held[live]
        got.append(to)
    return tuple(got)


def _values64(rows, heads, dim):
    """The values of e2m1 rows from the bits of their codes and scales."""
    n = heads * dim // 2
    code = torch.empty((*rows.shape[:-1], heads * dim), dtype=torch.int64, device=rows.device)
    code[..., 0::2], code[..., 1::2] = rows[..., :n].long() % 16, rows[..., :n].long() // 16
    sign, e, m = 1 - 2 * (code // 8).double(), code // 2 % 4, (code % 2).double()
    x = sign * torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2((e - 1).double()))
    b = rows[..., n:n + heads * dim // 16].long()
    e, m = b // 8 % 16, (b % 8).double()
    scale = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2((e - 7).double()))
    return (x.unflatten(-1, (-1, 16)) * scale[..., None]).reshape(*rows.shape[:-1], heads, dim)


def _exact_attention(st, dev):
    case = st["case"]
    step, heads, dim = case["op"] == "step", case["heads"], case["dim"]
    window = case["window"] or 1 << 60
    out = torch.zeros(st["query"].shape, dtype=torch.float64, device=dev)
    lse = torch.full(st["query"].shape[:2], -math.inf, dtype=torch.float64, device=dev)
    first = 0
    for i, (n, fresh) in enumerate(zip(st["lens_host"], st["new_host"])):
        row0 = i if step else first
        first += fresh
        if not n:
            continue
        low = max(0, n - fresh - window + 1)  # tokens before this are seen as sinks only
        j = torch.tensor([t for t in range(n) if t >= low or t < case["sinks"]], device=dev)
        flat = st["tables"][i][j.div(case["block"], rounding_mode="floor")] * case["block"] + j.remainder(case["block"])
        k_all = _values64(st["key"].flatten(0, 1)[flat], heads, dim)
        v_all = _values64(st["value"].flatten(0, 1)[flat], heads, dim)
        for r0 in range(0, fresh, 512):
            r1 = min(fresh, r0 + 512)
            p = torch.arange(n - fresh + r0, n - fresh + r1, device=dev)[:, None]
            seen = (j <= p) & ((p - j < window) | (j < case["sinks"]))
            for head in range(heads * case["group"]):
                kv_head = head // case["group"]
                q = st["query"][row0 + r0:row0 + r1, head].double()
                s = (q @ k_all[:, kv_head].T) * st["scale"]
                logs = torch.logsumexp(torch.where(seen, s, -math.inf), dim=1)
                weight = torch.where(seen, torch.exp(s - logs[:, None]), 0.0)
                out[row0 + r0:row0 + r1, head] = weight @ v_all[:, kv_head]
                lse[row0 + r0:row0 + r1, head] = logs
    return out, lse
