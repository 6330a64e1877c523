"""rotate_tokens, append_tokens and read_tokens against 64-bit arithmetic:
types, layouts of pairs, head dims, strides, padding, caches of 16, 8 and 4
bits, values at the ends of their range, streams and graphs."""
from __future__ import annotations

import math

import pytest
import torch

import token_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def rows_of(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def places(rows, most, seed):
    return torch.randint(0, most, (rows,), generator=torch.Generator().manual_seed(seed + 1))


# ---------------------------------------------------------------------------
# rotation
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim,rotary", [(8, 2), (8, 8), (64, 64), (80, 80), (96, 48), (112, 84), (128, 128), (128, 32),
                                        (128, 50), (256, 256), (256, 192), (24, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation(ops, dev, dtype, dim, rotary, interleaved):
    x = rows_of((13, 5, dim), dtype, dim + rotary)
    at = places(13, 700, dim)
    table = ops.rotary_table(700, rotary, base=5000.0)
    for transpose in (False, True):
        want, bound = oracle.rotate(x, at, table, interleaved=interleaved, transpose=transpose)
        got = ops.rotate_tokens(x.to(dev), at.to(dev), table.to(dev), interleaved=interleaved, transpose=transpose,
                                check=True)
        oracle.check_rows(got.cpu(), want, bound, dtype)
        assert torch.equal(got.cpu()[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("rows,heads", [(1, 1), (1, 40), (3, 7), (1000, 3), (20000, 2)])
def test_rotation_sizes(ops, dev, rows, heads):
    x = rows_of((rows, heads, 64), BF16, rows)
    at = places(rows, 50, rows)
    table = ops.rotary_table(50, 64)
    want, bound = oracle.rotate(x, at, table)
    oracle.check_rows(ops.rotate_tokens(x.to(dev), at.to(dev), table.to(dev), check=True).cpu(), want, bound, BF16)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [80, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_in_place_and_strides(ops, dev, dtype, dim, interleaved):
    both = rows_of((33, 9, dim), dtype, dim).to(dev)
    x = both[:, 2:7]
    at = places(33, 90, dim)
    at[[0, 31]] = -1  # padding
    table = ops.rotary_table(90, dim).to(dev)
    want, bound = oracle.rotate(x.cpu(), at.clamp(min=0), table.cpu(), interleaved=interleaved)
    want[[0, 31]], bound[[0, 31]] = x.cpu().double()[[0, 31]], 0.0
    before = both.clone()
    # heads outside, rows within in memory
    out = torch.full((5, 33, dim), 7.0, dtype=dtype, device=dev).transpose(0, 1)
    ops.rotate_tokens(x, at.to(dev), table, interleaved=interleaved, out=out, check=True)
    assert (out[[0, 31]] == 7).all() and torch.equal(both, before)
    live = [r for r in range(33) if r not in (0, 31)]
    oracle.check_rows(out.cpu()[live], want[live], bound[live], dtype)
    got = ops.rotate_tokens(x, at.to(dev), table, interleaved=interleaved, out=x, check=True)
    assert got is x
    oracle.check_rows(x.cpu(), want, bound, dtype)
    assert torch.equal(both[:, :2], before[:, :2]) and torch.equal(both[:, 7:], before[:, 7:])


def test_rotation_of_every_pair_form_agrees_bit_for_bit_with_plain_rounding(ops, dev):
    x, at = rows_of((50, 4, 128), F32, 3).to(dev), places(50, 300, 3).to(dev)
    table = ops.rotary_table(300, 96).to(dev)
    c, s = table[at][:, None, :48], table[at][:, None, 48:]
    a, b = x[..., :48], x[..., 48:96]
    want = torch.cat([a * c - b * s, b * c + a * s, x[..., 96:]], -1)
    assert torch.equal(ops.rotate_tokens(x, at, table, check=True), want)
    a, b = x[..., 0:96:2], x[..., 1:96:2]
    want = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., 96:]], -1)
    assert torch.equal(ops.rotate_tokens(x, at, table, interleaved=True, check=True), want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_transpose_is_the_gradient(ops, dev, interleaved):
    x, g = rows_of((6, 2, 32), F32, 1), rows_of((6, 2, 32), F32, 2)
    at = places(6, 40, 1)
    table = ops.rotary_table(40, 24, scaling="yarn", factor=8.0, original_positions=16)

    def turn(v, **kw):
        return ops.rotate_tokens(v.to(dev), at.to(dev), table.to(dev), interleaved=interleaved, check=True,
                                 **kw).cpu().double()

    grad = turn(g, transpose=True)
    # differences: the rotation is linear, so a step of 1 has no error but rounding (2^-23 of some products)
    for d in range(32):
        step = torch.zeros((6, 2, 32))
        step[..., d] = 1.0
        slope = (turn(x + step) - turn(x)) * g.double()
        size = (turn(x + step).abs() + turn(x).abs()) * g.double().abs()
        err = (slope.sum(-1) - grad[..., d]).abs()
        assert (err <= 2.0 ** -21 * (size.sum(-1) + 32)).all()
    want, bound = oracle.rotate(g, at, table, interleaved=interleaved, transpose=True)
    assert ((grad - want).abs() <= bound + oracle.rounding(want, F32)).all()


def test_transpose_leads_back(ops, dev):
    x, at = rows_of((100, 3, 128), F32, 4).to(dev), places(100, 1 << 20, 4).to(dev)
    table = ops.rotary_table(1 << 20, 128, base=1e6, device=dev)
    there = ops.rotate_tokens(x, at, table, check=True)
    back = ops.rotate_tokens(there, at, table, transpose=True, out=there, check=True)
    # r: a pair's norm, at most 6.5 here.  Each way rounds by 2.41 r 2^-24 per value, the first one's error turns with
    # the pair (1.41 times), and c^2 + s^2 is off by 1.41 * 2^-24: 7.3 r 2^-24 in all
    assert x.abs().max() < 4.6 and (back - x).abs().max() <= 48 * 2.0 ** -24


def test_rotation_reports_a_bad_position_and_goes_on(ops, dev):
    x = rows_of((5, 2, 64), F16, 5).to(dev)
    table = ops.rotary_table(10, 64).to(dev)
    out = torch.full_like(x, 3.0)
    with pytest.raises(IndexError, match="10 is out of range"):
        ops.rotate_tokens(x, torch.tensor([0, 1, 10, 3, 9], device=dev), table, out=out, check=True)
    assert (out[2] == 3).all()
    want, bound = oracle.rotate(x.cpu(), torch.tensor([0, 1, 0, 3, 9]), table.cpu())
    oracle.check_rows(out.cpu()[[0, 1, 3, 4]], want[[0, 1, 3, 4]], bound[[0, 1, 3, 4]], F16)


def test_infinities_turn_with_their_pair_only(ops, dev):
    x = rows_of((1, 1, 64), F32, 6)
    x[0, 0, 3] = math.inf
    x[0, 0, 40:48] = torch.tensor([math.nan] * 8)
    table = ops.rotary_table(10, 32)
    got = ops.rotate_tokens(x.to(dev), torch.tensor([7], device=dev), table.to(dev), check=True).cpu()[0, 0]
    odd = ~torch.isfinite(got)
    assert odd.nonzero().view(-1).tolist() == [3, 19, *range(40, 48)]  # beyond the rotary dims they stay


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def cache_of(kind, slots, block, heads, dim, dev, layout="nhd"):
    """A cache plane whose bytes are all 0x5a, and a function that gives its token rows."""
    if kind == "e2m1":
        size = -(-heads * dim * 9 // 256) * 16
        if layout == "merged":
            both = torch.full((slots, block, 2, size), 0x5a, dtype=torch.uint8, device=dev)
            return both[:, :, 0], both[:, :, 1]
        return tuple(torch.full((slots, block, size), 0x5a, dtype=torch.uint8, device=dev) for _ in range(2))
    size = torch.empty((), dtype=kind).element_size()

    def new(*shape):
        return torch.full((*shape[:-1], shape[-1] * size), 0x5a, dtype=torch.uint8, device=dev).view(kind)

    if layout == "hnd":
        return tuple(new(slots, heads, block, dim).transpose(1, 2) for _ in range(2))
    if layout == "merged":
        both = new(slots, block, 2, heads, dim)
        return both[:, :, 0], both[:, :, 1]
    return tuple(new(slots, block, heads, dim) for _ in range(2))


def stored(cache, slots):
    rows = cache.flatten(0, 1) if cache.is_contiguous() else cache.reshape(-1, *cache.shape[2:])
    return rows.view(torch.uint8)[slots] if cache.dtype == E4M3 else rows[slots]


def check_stored(cache, mapping, want, bound, kind, factor):
    """The rows named by mapping hold want; every other byte is as it was."""
    host = cache.cpu()
    block = host.shape[1]
    live = mapping >= 0
    got = stored(host.contiguous(), mapping[live])
    if kind == "e2m1":
        n = want.shape[1] * want.shape[2] * 9 // 16
        oracle.check_e2m1(got, want[live], bound[live], factor)
        left = host.contiguous().flatten(0, 1)
        assert (left[:, n:] == 0x5a).all()
    elif kind == E4M3:
        oracle.check_e4m3(got.view(E4M3), want[live], bound[live], factor)
    else:
        oracle.check_rows(got, want[live], bound[live], kind)
    rest = torch.ones(host.shape[0] * block, dtype=torch.bool)
    rest[mapping[live]] = False
    bytes_of = host.contiguous().view(torch.uint8).flatten(0, 1)
    assert (bytes_of[rest] == 0x5a).all()


def append(ops, dev, *, dtype, cache, rows=37, heads=2, group=3, dim=64, rotary=None, block=16, layout="nhd",
           interleaved=False, pad=(), seed=0, query=True, table=True, scales=(1.0, 1.0), magnitude=1.0):
    kind = dtype if cache is None else cache
    rotary = dim if rotary is None else rotary
    both = rows_of((rows, heads * (group + 2), dim), F32, seed).mul_(magnitude).to(dtype)
    q, k, v = both.split([heads * group, heads, heads], 1)
    on = both.to(dev).split([heads * group, heads, heads], 1)
    slots = -(-rows // block) + 2
    order = torch.randperm(slots * block, generator=torch.Generator().manual_seed(seed + 2))
    mapping = order[:rows].clone()
    mapping[list(pad)] = -1
    at = places(rows, 300, seed)
    turn = ops.rotary_table(300, rotary) if table else None
    kc, vc = cache_of(kind, slots, block, heads, dim, dev, layout)
    kw = dict(positions=at.to(dev), table=turn.to(dev), interleaved=interleaved) if table else {}
    out = None
    if query:
        out = torch.full(q.shape, 9.0, dtype=dtype, device=dev)
        kw.update(query=on[0], query_out=out)
    if kind != dtype:
        kw.update(key_scale=scales[0], value_scale=scales[1])
    got = ops.append_tokens(on[1], on[2], kc, vc, mapping.to(dev), check=True, **kw)
    assert got is out
    live = mapping >= 0
    if table:
        want_k, bound = oracle.rotate(k, at, turn, interleaved=interleaved)
        want_q, q_bound = oracle.rotate(q, at, turn, interleaved=interleaved)
    else:
        want_k, bound = k.double(), torch.zeros(k.shape, dtype=torch.float64)
    if query:
        oracle.check_rows(out.cpu()[live], want_q[live], q_bound[live], dtype)
        assert (out.cpu()[~live] == 9).all()
    zero = torch.zeros(v.shape, dtype=torch.float64)
    if layout == "merged":  # each plane is checked by itself: the other one lies between
        kc, vc = kc.contiguous(), vc.contiguous()
    check_stored(kc, mapping, want_k, bound, kind, scales[0])
    check_stored(vc, mapping, v.double(), zero, kind, scales[1])


CACHES = [None, E4M3, "e2m1"]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("rows", [1, 2, 37, 300])
def test_append(ops, dev, dtype, cache, rows):
    append(ops, dev, dtype=dtype, cache=cache, rows=rows, seed=rows)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim,rotary", [(32, 32), (64, 32), (96, 72), (128, 128), (128, 100), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_head_dims(ops, dev, cache, dim, rotary, interleaved):
    append(ops, dev, dtype=BF16, cache=cache, dim=dim, rotary=rotary, interleaved=interleaved, seed=dim)


@pytest.mark.parametrize("cache", [None, E4M3])
@pytest.mark.parametrize("dim", [16, 48, 80, 112, 240])
def test_append_head_dims_of_sixteen(ops, dev, cache, dim):
    append(ops, dev, dtype=F16, cache=cache, dim=dim, seed=dim)


def test_append_head_dims_of_eight(ops, dev):
    append(ops, dev, dtype=F16, cache=None, dim=24, seed=1)
    append(ops, dev, dtype=BF16, cache=None, dim=200, rotary=8, seed=2)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,group", [(1, 1), (1, 8), (3, 5), (8, 4), (7, 1), (40, 1)])
def test_append_heads(ops, dev, cache, heads, group):
    append(ops, dev, dtype=BF16, cache=cache, heads=heads, group=group, rows=11, seed=heads)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("block", [1, 3, 16, 48, 257])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "merged"])
def test_append_blocks_and_layouts(ops, dev, cache, block, layout):
    if cache == "e2m1" and layout == "hnd":
        layout = "nhd"
    append(ops, dev, dtype=F16, cache=cache, block=block, layout=layout, seed=block)


@pytest.mark.parametrize("cache", CACHES)
def test_append_padding(ops, dev, cache):
    append(ops, dev, dtype=BF16, cache=cache, pad=(0, 5, 6, 36), seed=3)
    append(ops, dev, dtype=BF16, cache=cache, rows=3, pad=(0, 1, 2), seed=4)


@pytest.mark.parametrize("cache", CACHES)
def test_append_without_rotation_or_query(ops, dev, cache):
    append(ops, dev, dtype=F16, cache=cache, table=False, query=False, seed=5)
    append(ops, dev, dtype=F16, cache=cache, query=False, seed=6)


@pytest.mark.parametrize("cache", [E4M3, "e2m1"])
@pytest.mark.parametrize("scales", [(0.0625, 0.25), (0.013, 3.7)])
@pytest.mark.parametrize("magnitude", [1.0, 300.0, 1e-4])
def test_append_scales(ops, dev, cache, scales, magnitude):
    append(ops, dev, dtype=BF16, cache=cache, scales=scales, magnitude=magnitude, seed=7)


def test_append_query_in_place(ops, dev):
    both = rows_of((20, 8, 64), BF16, 8).to(dev)
    before = both.clone()
    at = places(20, 60, 8).to(dev)
    table = ops.rotary_table(60, 64).to(dev)
    kc, vc = cache_of(BF16, 4, 16, 2, 64, dev)
    q = both[:, :4]
    assert ops.append_tokens(both[:, 4:6], both[:, 6:], kc, vc, torch.arange(20, device=dev), positions=at, table=table,
                             query=q, query_out=q, check=True) is q
    want, bound = oracle.rotate(before[:, :4].cpu(), at.cpu(), table.cpu())
    oracle.check_rows(q.cpu(), want, bound, BF16)
    assert torch.equal(both[:, 4:], before[:, 4:])
    assert torch.equal(stored(vc, torch.arange(20, device=dev)), before[:, 6:])


@pytest.mark.parametrize("cache", CACHES)
def test_append_reports_bad_rows_and_goes_on(ops, dev, cache):
    kind = F16 if cache is None else cache
    k, v = rows_of((4, 2, 64), F16, 9), rows_of((4, 2, 64), F16, 10)
    at = torch.tensor([0, 1, 2, 3])
    table = ops.rotary_table(4, 64)
    for mapping, positions, bad in (([3, 64, 5, 9], [0, 1, 2, 3], 64), ([3, 4, 5, 9], [0, 4, 2, 3], 4),
                                    ([3, 4, 5, 9], [0, -1, 2, 3], -1)):
        kc, vc = cache_of(kind, 4, 16, 2, 64, dev)
        with pytest.raises(IndexError, match=f"{bad} is out of range"):
            ops.append_tokens(k.to(dev), v.to(dev), kc, vc, torch.tensor(mapping, device=dev),
                              positions=torch.tensor(positions, device=dev), table=table.to(dev), check=True)
        want, bound = oracle.rotate(k, at, table)
        left = torch.tensor([m if r != 1 else -1 for r, m in enumerate(mapping)])
        check_stored(kc, left, want, bound, kind, 1.0)
        check_stored(vc, left, v.double(), torch.zeros_like(bound), kind, 1.0)


def test_four_bit_values_at_the_ends_of_their_range(ops, dev):
    v = torch.zeros((6, 1, 32), dtype=BF16)
    v[0, 0, :3] = torch.tensor([math.inf, -5.0, 448.0])
    v[1, 0, 16:18] = torch.tensor([math.nan, 1.0])
    v[2, 0, :4] = torch.tensor([1e30, -1e30, 2688.0, 1344.0])
    v[3, 0, :2] = torch.tensor([1e-30, -1e-30])
    v[4, 0, :3] = torch.tensor([2.0 ** -9 * 6, 2.0 ** -9, -2.0 ** -10])
    v[5, 0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 2) * torch.tensor([1.0] * 8 + [-1.0] * 8)
    kc, vc = cache_of("e2m1", 1, 8, 1, 32, dev)
    ops.append_tokens(v.to(dev), v.to(dev), kc, vc, torch.arange(6, device=dev), check=True)
    assert torch.equal(kc, vc)
    got = ops.read_tokens(vc, torch.arange(6, device=dev), head_dim=32, dtype=F32, check=True).cpu()[:, 0]
    assert got[0, :3].tolist() == [2688.0, 0.0, 448.0] and (got[0, 3:] == 0).all()  # 448 is one unit, 5 none
    assert torch.isnan(got[1, 16:]).all() and (got[1, :16] == 0).all()
    assert got[2, :4].tolist() == [2688.0, -2688.0, 2688.0, 1344.0]
    assert (got[3] == 0).all()
    assert got[4, :3].tolist() == [2.0 ** -9 * 6, 2.0 ** -9, -2.0 ** -10]
    ties = torch.tensor([0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0])  # to even codes
    assert torch.equal(got[5, :8], ties) and torch.equal(got[5, 8:16], -ties)


def test_quotients_are_rounded_as_divisions(ops, dev):
    # every pair of a bf16 value and a scale in a range of exponents: the code is that of the rounded quotient
    v = torch.randn((4096, 1, 256), generator=torch.Generator().manual_seed(1)).mul_(
        torch.exp2(torch.randint(-12, 9, (4096, 1, 1), generator=torch.Generator().manual_seed(2)).float())).to(BF16)
    factor = 0.37
    kc, vc = cache_of("e2m1", 256, 16, 1, 256, dev)
    ops.append_tokens(v.to(dev), v.to(dev), kc, vc, torch.arange(4096, device=dev), key_scale=factor, value_scale=1.0,
                      check=True)
    for cache, f in ((kc, factor), (vc, 1.0)):
        f = torch.tensor(f, device=dev)
        g = v.to(dev).float().view(4096, 16, 16)
        scale = (g.abs().amax(-1) / (6 * f)).clamp(max=448).to(E4M3)
        got, held = oracle.unpack(cache.cpu().flatten(0, 1), 1, 256)
        assert torch.equal(held.view(4096, 16), scale.cpu().double())
        unit = (scale.float() * f)[..., None]
        y = torch.where(unit > 0, g / unit, 0.0).abs()
        code = sum((y > t if i % 2 == 0 else y >= t).long() for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
        want = oracle.E2M1[code.cpu()] * torch.where(g.cpu() < 0, -1.0, 1.0)
        assert torch.equal(got.view(4096, 16, 16), want)


# ---------------------------------------------------------------------------
# reading back
# ---------------------------------------------------------------------------


def test_every_code_and_scale(ops, dev):
    # 256 tokens, one per scale byte, each with all bytes of codes (512 values: 2 heads of 256)
    rows = torch.zeros((1, 256, -(-512 * 9 // 256) * 16), dtype=torch.uint8)
    rows[0, :, :256] = torch.arange(256, dtype=torch.uint8)
    rows[0, :, 256:288] = torch.arange(256, dtype=torch.uint8)[:, None]
    at = torch.arange(256)
    for dtype in (F16, BF16, F32):
        got = ops.read_tokens(rows.to(dev), at.to(dev), head_dim=256, dtype=dtype, check=True).cpu()
        want = oracle.values(rows[0], 2, 256)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.double().nan_to_num(), want.nan_to_num())  # every value has at most 6 bits


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads,dim", [(1, 16), (3, 80), (8, 128), (2, 256)])
def test_read_e4m3(ops, dev, dtype, heads, dim):
    plane = (rows_of((5, 16, heads, dim), F32, dim) * 20).to(E4M3)
    mapping = torch.randperm(80, generator=torch.Generator().manual_seed(dim))[:50]
    mapping[[3, 49]] = -1
    out = torch.full((50, heads, dim), 5.0, dtype=dtype, device=dev)
    got = ops.read_tokens(plane.to(dev), mapping.to(dev), scale=0.3, out=out, check=True)
    assert got is out
    live = mapping >= 0
    want = plane.flatten(0, 1).double()[mapping.clamp(min=0)] * 0.3
    assert (out.cpu()[~live] == 5).all()
    oracle.check_rows(out.cpu()[live], want[live], want[live].abs() * 2.0 ** -23, dtype)


@pytest.mark.parametrize("heads,dim", [(1, 32), (3, 96), (8, 128), (5, 256), (7, 32)])
def test_read_e2m1(ops, dev, heads, dim):
    x = rows_of((80, heads, dim), F32, dim)
    rows = oracle.pack(x, heads, dim).view(5, 16, -1)
    mapping = torch.randperm(80, generator=torch.Generator().manual_seed(dim))[:50]
    mapping[[0, 20]] = -1
    out = torch.full((50, heads, dim), 5.0, dtype=F32, device=dev)
    ops.read_tokens(rows.to(dev), mapping.to(dev), head_dim=dim, scale=0.3, out=out, check=True)
    live = mapping >= 0
    want = oracle.values(rows.flatten(0, 1)[mapping.clamp(min=0)], heads, dim, 0.3)
    assert (out.cpu()[~live] == 5).all()
    oracle.check_rows(out.cpu()[live], want[live], want[live].abs() * 2.0 ** -22, F32)


@pytest.mark.parametrize("heads,dim,kind", [(1, 16, E4M3), (2, 16, E4M3), (1, 32, "e2m1"), (13, 256, "e2m1"),
                                            (13, 256, E4M3)])
def test_read_of_many_rows(ops, dev, heads, dim, kind):
    g = torch.Generator(device=dev).manual_seed(dim)
    mapping = torch.randperm(40 * 160, generator=g, device=dev)[:6001]
    if kind == E4M3:
        plane = torch.randn((160, 40, heads, dim), generator=g, device=dev).to(E4M3)
        want = plane.float().flatten(0, 1)[mapping]
    else:
        plane = torch.randint(0, 256, (160, 40, ops.e2m1_row_bytes(heads, dim)), generator=g, device=dev,
                              dtype=torch.uint8)
        plane[:, :, heads * dim // 2:] &= 0x3f  # scales from 0 to 1.9
        want = oracle.values(plane.flatten(0, 1)[mapping].cpu(), heads, dim).float().to(dev)
    for offset in (0, 8):  # places in steps of 32 bytes, and of 16
        out = torch.empty(want.numel() + 8, dtype=F16, device=dev)[offset:offset + want.numel()].view(want.shape)
        ops.read_tokens(plane, mapping, head_dim=dim, out=out, check=True)
        assert torch.equal(out, want.half())


@pytest.mark.parametrize("four", [False, True])
def test_read_reports_a_bad_slot_and_goes_on(ops, dev, four):
    plane = torch.zeros((2, 4, 80), dtype=torch.uint8, device=dev) if four else \
        torch.zeros((2, 4, 1, 128), device=dev).to(E4M3)
    out = torch.ones((3, 1, 128), dtype=F16, device=dev)
    with pytest.raises(IndexError, match="8 is out of range"):
        ops.read_tokens(plane, torch.tensor([7, 8, 0], device=dev), head_dim=128, out=out, check=True)
    assert (out[1] == 1).all() and (out[[0, 2]] == 0).all()


# ---------------------------------------------------------------------------
# places, streams, graphs
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["e2m1", F16])
def test_places_past_four_gigabytes(ops, dev, cache):
    heads, dim, block = 8, 128, 16
    size = 576 if cache == "e2m1" else 2048
    slots = (1 << 32) // (size * block) + 5
    planes = [torch.empty((slots, block, size), dtype=torch.uint8, device=dev) for _ in range(2)]
    if cache != "e2m1":
        planes = [p.view(F16).view(slots, block, heads, dim) for p in planes]
    k, v = rows_of((2, heads, dim), F16, 1), rows_of((2, heads, dim), F16, 2)
    mapping = torch.tensor([slots * block - 1, 17], device=dev)
    ops.append_tokens(k.to(dev), v.to(dev), *planes, mapping, check=True)
    for plane, x in zip(planes, (k, v)):
        rows = plane.view(-1, *plane.shape[2:])[mapping]
        if cache == "e2m1":
            oracle.check_e2m1(rows.cpu(), x.double(), torch.zeros(x.shape, dtype=torch.float64), 1.0)
            got = ops.read_tokens(plane, mapping, head_dim=dim, dtype=F32, check=True)
            assert torch.equal(got.cpu().double(), oracle.values(rows.cpu(), heads, dim))
        else:
            assert torch.equal(rows.cpu(), x)


def test_another_stream_and_a_graph(ops, dev):
    k = rows_of((30, 2, 64), BF16, 1).to(dev)
    at, mapping = places(30, 100, 1).to(dev), torch.randperm(48, generator=torch.Generator().manual_seed(1))[:30].to(dev)
    table = ops.rotary_table(100, 64).to(dev)
    want_k, want_v = cache_of("e2m1", 3, 16, 2, 64, dev)
    q = rows_of((30, 4, 64), BF16, 2).to(dev)
    kw = dict(positions=at, table=table, query=q, check=False)
    want_q = ops.append_tokens(k, k, want_k, want_v, mapping, **kw)
    want = ops.read_tokens(want_k, mapping, head_dim=64, check=True)
    stream = torch.cuda.Stream(dev)
    kc, vc = cache_of("e2m1", 3, 16, 2, 64, dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        got_q = ops.append_tokens(k, k, kc, vc, mapping, **kw)
        got = ops.read_tokens(kc, mapping, head_dim=64, check=False)
    stream.synchronize()
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v) and torch.equal(got, want) and torch.equal(got_q, want_q)
    live_k, out_q = k.clone(), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    kw["query_out"] = out_q
    with torch.cuda.graph(graph):
        ops.append_tokens(live_k, live_k, kc, vc, mapping, **kw)
        back = ops.rotate_tokens(out_q, at, table, transpose=True, check=False)
        read = ops.read_tokens(kc, mapping, head_dim=64, check=False)
    for seed in (3, 4):
        live_k.copy_(rows_of((30, 2, 64), BF16, seed))
        graph.replay()
        torch.cuda.synchronize()
        ops.append_tokens(live_k, live_k, want_k, want_v, mapping, positions=at, table=table, check=True)
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
        assert torch.equal(read, ops.read_tokens(want_k, mapping, head_dim=64, check=True))
        # two bf16 roundings of values to 4.5 or so
        assert (back.float() - q.float()).abs().max() <= 8 * 2.0 ** -8


def test_another_device(ops):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    dev = torch.device("cuda", 1)
    append(ops, dev, dtype=BF16, cache="e2m1")


def test_nothing_to_do(ops, dev):
    none = torch.zeros((0,), dtype=torch.int64, device=dev)
    k = torch.zeros((0, 2, 64), dtype=F16, device=dev)
    kc, vc = cache_of("e2m1", 1, 16, 2, 64, dev)
    assert ops.append_tokens(k, k, kc, vc, none, check=True) is None
    assert ops.read_tokens(kc, none, head_dim=64, check=True).shape == (0, 2, 64)
    assert ops.rotate_tokens(k, none, ops.rotary_table(3, 64).to(dev), check=True).shape == k.shape
    # a cache without blocks: every slot is out of range, padding is not
    empty = torch.zeros((0, 16, 80), dtype=torch.uint8, device=dev)
    one = torch.ones((1, 2, 64), dtype=F16, device=dev)
    ops.append_tokens(one, one, empty, empty.clone(), torch.tensor([-1], device=dev), check=True)
    with pytest.raises(IndexError):
        ops.append_tokens(one, one, empty, empty.clone(), torch.tensor([0], device=dev), check=True)


def test_refusals(ops, dev):
    k, at = torch.zeros((4, 2, 64), dtype=F16, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    table = ops.rotary_table(8, 64).to(dev)
    kc, vc = cache_of(F16, 4, 16, 2, 64, dev)
    four = cache_of("e2m1", 4, 16, 2, 64, dev)
    good = dict(positions=at, table=table, query=k, query_out=torch.empty_like(k))
    ops.append_tokens(k, k, kc, vc, torch.arange(4, device=dev), check=True, **good)
    merged = torch.zeros((4, 16, 2, 2, 64), dtype=F16, device=dev)
    ops.append_tokens(k, k, merged[:, :, 1], merged[:, :, 0], at + 63, check=True)
    for args, kw, match in (
            ((k, k[:3], kc, vc, at), {}, "share shape"),
            ((k, k, kc, four[1], at), {}, "share shape"),
            ((k, k, kc.float(), vc.float(), at), {}, "incorrect dtype"),
            ((k, k, kc[:, :, :1], vc[:, :, :1], at), {}, "must be"),
            ((k, k, four[0][:, :, :64], four[1][:, :, :64], at), {}, "no heads"),
            ((k[..., :48].contiguous(), k[..., :48].contiguous(), *four, at), {}, "out of range"),
            ((k, k, kc, vc, at[:3]), {}, "one entry"),
            ((k, k, kc, vc, at.int()), {}, "incorrect dtype"),
            ((k, k, kc, vc, at), dict(positions=at), "go together"),
            ((k, k, kc, vc, at), dict(query=k), "needs positions"),
            ((k, k, kc, vc, at), dict(query_out=k), "needs a query"),
            ((k, k, kc, vc, at), dict(key_scale=2.0), "belong to"),
            ((k, k, *four, at), dict(key_scale=0.0), "positive"),
            ((k, k, *four, at), dict(value_scale=math.nan), "positive"),
            ((k, k, kc, kc, at), {}, "share memory"),
            ((k, k, kc[:2], kc[1:3], at), {}, "share memory"),
            ((k, k, kc.expand(2, 4, 16, 2, 64)[:, 0], vc[:2], at), {}, "share memory"),
            ((kc[0][:4], k, kc, vc, at), {}, "overlap the rows"),
            ((k, k, kc, vc, at), dict(good, table=table[:, :3]), "contiguous"),
            ((k, k, kc, vc, at), dict(good, table=table.half()), "incorrect dtype"),
            ((k, k, kc, vc, at), dict(good, table=ops.rotary_table(8, 66).to(dev)), "at most head_dim"),
            ((k, k, kc, vc, at), dict(good, query_out=torch.empty((4, 2, 64), device=dev)), "incorrect dtype"),
            ((k, k, kc, vc, at), dict(good, query=k.expand(4, 2, 64)[:, :1].expand(4, 3, 64), query_out=k[:, :1].expand(4, 3, 64)),
             "share memory")):
        with pytest.raises((ValueError, TypeError), match=match):
            ops.append_tokens(*args, **kw)
    x = torch.zeros((6, 2, 64), dtype=F16, device=dev)
    for args, kw, match in (((x.double(), at, table), {}, "incorrect dtype"), ((x[0], at, table), {}, "must be"),
                            ((x, at, table), {}, "one entry"), ((x[:4], at, table), dict(out=x[1:5]), "overlap"),
                            ((x[:4, :, ::2], at, table), {}, "contiguous"), ((x[:4, :, :12], at, table), {}, "multiples"),
                            ((x[:4], at, table.cpu()), {}, "on cuda")):
        with pytest.raises((ValueError, TypeError), match=match):
            ops.rotate_tokens(*args, **kw)
    for args, kw, match in (((four[0], at), {}, "needs head_dim"), ((kc, at), {}, "incorrect dtype"),
                            ((four[0], at), dict(head_dim=96), "no heads"),
                            ((four[0], at), dict(head_dim=64, dtype=torch.int8), "incorrect dtype"),
                            ((four[0], at), dict(head_dim=64, out=k[:3]), "must be a contiguous")):
        with pytest.raises((ValueError, TypeError), match=match):
            ops.read_tokens(*args, **kw)


class Rotated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, x, positions, table, interleaved):
        ctx.save_for_backward(positions, table)
        ctx.ops, ctx.interleaved = ops, interleaved
        return ops.rotate_tokens(x, positions, table, interleaved=interleaved, check=True)

    @staticmethod
    def backward(ctx, grad):
        return (None, ctx.ops.rotate_tokens(grad.contiguous(), *ctx.saved_tensors, interleaved=ctx.interleaved,
                                            transpose=True, check=True), None, None, None)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_through_an_autograd_function_and_refused_without(ops, dev, interleaved):
    """The loss <w, y> + |y|^2 / 2 of y = R x changes over a step d by exactly
    <gradient, d> + |d|^2 / 2.  In fp32 a value of y is off by at most 4 half steps of
    |x1| + |x2| (two products, a sum, the table), which count |w| + |y| times in the
    loss, and so does the gradient: over a head, whose sums hold every pair's, and for
    two losses, the gradient and lengths that the table keeps but for its rounding, 4
    times that.  The rest is in 64 bits."""
    x, step, w = (rows_of((33, 5, 64), F32, seed).to(dev) for seed in (1, 2, 3))
    at = places(33, 500, 4).to(dev)
    table = ops.rotary_table(500, 64, device=dev)
    x.requires_grad_()
    for out in (None, x.detach().clone()):
        with pytest.raises(RuntimeError, match="records no gradient"):
            ops.rotate_tokens(x, at, table, interleaved=interleaved, out=out)
    with torch.no_grad():
        assert not ops.rotate_tokens(x, at, table, interleaved=interleaved).requires_grad

    def loss(v):
        y = Rotated.apply(ops, v, at, table, interleaved).double()
        return (y * w.double()).sum() + (y ** 2).sum() / 2

    (grad,) = torch.autograd.grad(loss(x), x)
    with torch.no_grad():
        there = x + step
        moved = there.double() - x.double()
        want = (grad.double() * moved).sum() + (moved ** 2).sum() / 2
        size = (x.abs() + there.abs()).double()
        bound = 4 * 4 * 2.0 ** -24 * (size.sum(-1) * (w.abs().double() + size).sum(-1)).sum()
        assert abs(loss(there) - loss(x) - want) <= bound
