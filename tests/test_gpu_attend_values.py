"""attend_step and attend_chunk where single values decide: infinities and NaN
at visible tokens, weights far below the largest."""
from __future__ import annotations

import math

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def place(b, s, t):
    """Page and offset of token t of sequence s."""
    block = b.key.shape[1]
    return b.tables[s, t // block], t % block


def offsets_of(b, dev):
    return torch.tensor([0] + b.new, device=dev).cumsum(0)


def attend(ops, dev, b, which, **kw):
    key, value = b.on(dev)
    query, tables, lens = b.query.to(dev), b.tables.to(dev), torch.tensor(b.lens, device=dev)
    lse = torch.empty(query.shape[:2], device=dev)
    kw = dict(window=b.window, sinks=b.sinks, lse=lse, check=True, **b.scales, **kw)
    if which == "step":
        out = ops.attend_step(query, key, value, tables, lens, **kw)
    else:
        out = ops.attend_chunk(query, offsets_of(b, dev), key, value, tables, lens, **kw)
    return out.cpu().double(), lse.cpu().double()


def agree(got, want, bound):
    """The same infinities and NaN, and every finite value within its bound."""
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    finite = torch.isfinite(want)
    err = (got - want).abs()[finite]
    assert (err <= bound[finite]).all(), (err / bound[finite]).max()


def plant(b, dims):
    """dims: (sequence, token, K/V head, dim, value) each."""
    for s, t, head, d, x in dims:
        page, off = place(b, s, t)
        b.value[page, off, head, d] = x


INF, NAN = math.inf, math.nan


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_step_of_one_infinite_token(ops, dev, dtype):
    b = oracle.Batch(lens=[1, 1], heads=1, group=2, dim=64, block=16, dtype=dtype, seed=1)
    plant(b, [(0, 0, 0, d, INF if d % 2 else -INF) for d in range(64)])
    out, _ = attend(ops, dev, b, "step")
    assert (out[0, :, 1::2] == INF).all() and (out[0, :, ::2] == -INF).all() and torch.isfinite(out[1]).all()


# magnitude 1: weights of one size; 12: weights to 2^-100 of the largest and less
@pytest.mark.parametrize("magnitude", [1.0, 12.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_step_with_infinite_values_at_visible_tokens(ops, dev, dtype, dim, magnitude):
    # one sequence over many runs of warps, and short ones within one
    b = oracle.Batch(lens=[3000, 40, 17, 500], heads=2, group=3, dim=dim, block=16, dtype=dtype, seed=dim,
                     magnitude=magnitude)
    marks = []
    for s, n in enumerate(b.lens):
        for i in range(0, dim, 5):
            marks.append((s, (i * 37) % n, i % 2, i, INF))
            marks.append((s, (i * 53 + 1) % n, i % 2, (i + 1) % dim, -INF))
        marks += [(s, 3, 0, 2, INF), (s, n - 1, 0, 2, -INF)]  # both: NaN
        marks += [(s, n // 2, 1, 3, NAN)]
    plant(b, marks)
    out, lse = attend(ops, dev, b, "step")
    _, (want, want_lse, bound, lse_bound) = b.expect(2.0 ** -11)
    agree(out, want, bound)
    assert ((lse - want_lse).abs() <= lse_bound).all()


def weak_batch(dtype, cache, sequences, tokens, new, heads, log2_gap, dim=64):
    """Per sequence one strong token (the first; its values are 0) and weak ones 2^-log2_gap of its weight (values 1).
    Returns the batch and the scale."""
    block = 16
    b = oracle.Batch(lens=[tokens] * sequences, new=[new] * sequences, heads=heads, group=1, dim=dim, block=block,
                     dtype=dtype, cache=cache, seed=2)
    b.scales = {}
    zero = torch.zeros((), dtype=b.key.dtype)
    b.key[:] = zero
    b.value[:] = torch.ones((), dtype=torch.float32).to(b.key.dtype)
    for s in range(sequences):
        page, off = place(b, s, 0)
        b.key[page, off, :, 0] = torch.tensor(16.0).to(b.key.dtype)
        b.value[page, off] = zero
    b.query = torch.zeros_like(b.query)
    b.query[:, :, 0] = 1.0
    return b, log2_gap * math.log(2.0) / 16.0


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
def test_step_keeps_weights_far_below_the_largest(ops, dev, dtype, cache):
    """2,000 tokens at 2^-26.3 of the first one's weight are all of the result."""
    b, scale = weak_batch(dtype, cache, sequences=40, tokens=2000, new=1, heads=8, log2_gap=26.3)
    out, lse = attend(ops, dev, b, "step", scale=scale)
    w = 2.0 ** -26.3
    want = 1999 * w / (1 + 1999 * w)
    # a weight to 2^-11 and the exponent's argument (26.3 in fp32, 2^-20), the result to its type's half step (fp16: of
    # a subnormal, 2^-25)
    eps = torch.finfo(dtype).eps / 2
    tol = want * (2.0 ** -11 + 2.0 ** -18 + eps) + (2.0 ** -25 if dtype == F16 else 0)
    assert ((out - want).abs() <= tol).all(), (out.min(), out.max(), want)
    assert ((lse - (26.3 * math.log(2.0) + math.log1p(1999 * w))).abs() <= 2.0 ** -17).all()


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunk_keeps_weights_far_below_the_largest(ops, dev, dtype, cache, dim):
    b, scale = weak_batch(dtype, cache, sequences=24, tokens=2000, new=8, heads=8, log2_gap=26.3, dim=dim)
    out, lse = attend(ops, dev, b, "chunk", scale=scale)
    w = 2.0 ** -26.3
    weak = torch.arange(1992, 2000, dtype=torch.float64).repeat(24).view(-1, 1)  # a row sees the first token and these
    want = (weak * w / (1 + weak * w)).unsqueeze(-1)
    # a weight to 2^-11 (bf16 2^-8) or, as an fp16 subnormal, to 2^-32 of the largest; the rest as for one token
    p_eps = 2.0 ** -8 if cache == BF16 else 2.0 ** -11
    steps = 0 if cache == BF16 else 2.0 ** -32
    tol = want * (p_eps + 2.0 ** -18 + torch.finfo(dtype).eps / 2) + weak.unsqueeze(-1) * steps
    if dtype == F16:
        tol = tol + 2.0 ** -25
    assert ((out - want).abs() <= tol).all(), (out.min(), out.max(), want)
    assert ((lse - (26.3 * math.log(2.0) + torch.log1p(weak * w))).abs() <= 2.0 ** -17).all()


def expect_chunk(b):
    return oracle.attention(b.query, b.key, b.value, b.tables.clamp(min=0), b.lens, b.new, window=b.window,
                            sinks=b.sinks, p_eps=2.0 ** -8 if b.key.dtype == BF16 else 2.0 ** -11, **b.scales)


@pytest.mark.parametrize("magnitude", [1.0, 12.0])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("dim", [48, 64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 20)])
def test_chunk_with_infinite_values(ops, dev, dtype, cache, dim, magnitude, window, sinks):
    """At tokens that all rows of a block see, some, or none; and every finite result as without them."""
    kw = dict(lens=[1700, 300, 300, 40], new=[3, 300, 130, 17], heads=2, group=3, dim=dim, block=16, dtype=dtype,
              cache=cache, seed=dim, magnitude=magnitude, window=window, sinks=sinks)
    b, clean = oracle.Batch(**kw), oracle.Batch(**kw)
    marks = []
    inf = NAN if cache == E4M3 else INF
    for s, (n, new) in enumerate(zip(b.lens, b.new)):
        low = max(0, n - new - window + 1) if window else 0  # no row sees what is before, but for the sinks
        span = n - low
        for i in range(0, dim, 7):
            marks.append((s, low + (i * 37) % span, i % 2, i, inf))
            marks.append((s, low + (i * 53 + 1) % span, i % 2, (i + 1) % dim, -inf))
        marks += [(s, low + 3, 0, 2, inf), (s, n - 1, 0, 2, -inf), (s, low + span // 2, 1, 3, NAN)]
        if window:
            marks += [(s, 0, 0, 5, inf), (s, sinks - 1, 1, 4, -inf)]
    plant(b, marks)
    out, lse = attend(ops, dev, b, "chunk")
    want, want_lse, bound, lse_bound = expect_chunk(b)
    agree(out, want, bound)
    agree(lse, want_lse, lse_bound)  # NaN where e4m3 keys of magnitude 12 x 16 are (above 448)
    same = attend(ops, dev, clean, "chunk")
    finite = torch.isfinite(out)
    assert torch.equal(out[finite], same[0][finite])
    assert torch.equal(lse.nan_to_num(nan=99.0), same[1].nan_to_num(nan=99.0))


@pytest.mark.parametrize("which", ["step", "chunk"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinite_value_of_weight_zero(ops, dev, which, dtype):
    """A key of -inf: the token's weight is 0, and 0 times an infinite value is NaN."""
    new = [1, 1] if which == "step" else [90, 3]
    b = oracle.Batch(lens=[90, 500], new=new, heads=1, group=2, dim=64, block=16, dtype=dtype, seed=4)
    b.query[:, :, 0] = b.query[:, :, 0].abs() + 0.5
    for s, t in ((0, 40), (1, 200), (1, 499)):
        page, off = place(b, s, t)
        b.key[page, off, 0, 0] = -INF
        b.value[page, off, 0, 7] = INF
    out, lse = attend(ops, dev, b, which)
    sees = torch.tensor([which == "step" or row >= 40 for row in range(b.query.shape[0])])
    assert torch.isnan(out[sees][:, :, 7]).all()
    out[:, :, 7] = torch.where(sees.view(-1, 1), 0.0, out[:, :, 7])
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3)])
def test_long_context_with_an_infinite_value(ops, dev, dtype, cache):
    """One value of an early token: 60,000 keys, 1,024 new tokens and a few of a second sequence."""
    n, block, heads, group, dim = 60_000, 16, 2, 4, 128
    g = torch.Generator(device=dev).manual_seed(3)
    pages = n // block
    key = torch.randn((2 * pages, block, heads, dim), generator=g, device=dev).to(cache)
    value = torch.randn((2 * pages, block, heads, dim), generator=g, device=dev).to(cache)
    query = torch.randn((1024 + 5, heads * group, dim), generator=g, device=dev).to(dtype)
    tables = torch.randperm(2 * pages, generator=g, device=dev).view(2, -1)
    offsets = torch.tensor([0, 1024, 1029], device=dev)
    lens = torch.tensor([n, n], device=dev)
    args = (query, offsets, key, value, tables, lens)
    clean = ops.attend_chunk(*args, check=True)
    bad = NAN if cache == E4M3 else INF
    value[tables[0, 100], 3, 1, 17] = bad    # all rows of the first sequence
    value[tables[0, -1], 8, 0, 20] = -bad    # the last eight tokens' rows
    value[tables[1, -1], 13, 1, 21] = bad    # the last three rows
    got = ops.attend_chunk(*args, check=True)
    want = clean.clone()
    want[:1024, group:, 17] = bad
    want[1016:1024, :group, 20] = -bad
    want[1026:, group:, 21] = bad
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=5.0), want.nan_to_num(nan=5.0))


@pytest.mark.parametrize("which", ["step", "chunk"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_values(ops, dev, which, dtype):
    """Averages of half the type's largest value are that value: sums of it do not overflow."""
    new = [1, 1, 1] if which == "step" else [400, 3, 5]
    b = oracle.Batch(lens=[400, 3000, 70], new=new, heads=2, group=2, dim=64, block=16, dtype=dtype, seed=6)
    most = torch.finfo(dtype).max / 2
    for s, n in enumerate(b.lens):
        for t in range(n):
            page, off = place(b, s, t)
            b.value[page, off, 0], b.value[page, off, 1] = most, -most
    out, _ = attend(ops, dev, b, which)
    # a weight's rounding (half a step at most), sums and the exponential (2^-20), the result's rounding
    tol = most * (torch.finfo(dtype).eps * 1.01 + 2.0 ** -20)
    assert ((out[:, :2] - most).abs() <= tol).all() and ((out[:, 2:] + most).abs() <= tol).all()


@pytest.mark.parametrize("dtype,p_eps", [(F16, 2.0 ** -21), (BF16, 2.0 ** -15)])
def test_step_weights_keep_more_than_their_type(ops, dev, dtype, p_eps):
    """Two values that nearly cancel: what is left shows the weights' last bits."""
    n = 64
    b = oracle.Batch(lens=[2] * n, heads=1, group=1, dim=64, block=16, dtype=dtype, seed=8)
    b.key.zero_()
    for s in range(n):
        page, _ = place(b, s, 0)
        b.key[page, 0, 0, 0] = 0.01 * (s + 1)
        b.value[page, 0], b.value[page, 1] = 1000.0, -1000.0
    b.query.zero_()
    b.query[:, :, 0] = 1.0
    out, _ = attend(ops, dev, b, "step", scale=1.0)
    want, _, bound, _ = oracle.attention(b.query, b.key, b.value, b.tables.clamp(min=0), b.lens, [1] * n, scale=1.0,
                                         p_eps=p_eps)
    agree(out, want, bound)
