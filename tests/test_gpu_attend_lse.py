"""The log of the softmax sum that attend_step and attend_chunk give, for any
sign of the scale and out of replayed graphs."""
from __future__ import annotations

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
# rounding of a probability on its way into the second product: bf16 chunks take bf16 ones, 2^-8
P_EPS = {"step": 2.0 ** -11, "chunk": 2.0 ** -8}


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def batch(which, dtype, cache, seed=1):
    lens, new = ([40, 900], [1, 1]) if which == "step" else ([340, 90], [40, 90])
    return oracle.Batch(lens=lens, new=new, heads=2, group=2, dim=64, block=16, dtype=dtype, cache=cache, seed=seed)


def arguments(ops, dev, b, which):
    key, value = b.on(dev)
    rest = (key, value, b.tables.to(dev), torch.tensor(b.lens, device=dev))
    if which == "step":
        return ops.attend_step, (b.query.to(dev), *rest)
    return ops.attend_chunk, (b.query.to(dev), torch.tensor([0] + b.new, device=dev).cumsum(0), *rest)


def check(b, which, out, lse, **kw):
    want, want_lse, bound, lse_bound = oracle.attention(b.query, b.key, b.value, b.tables.clamp(min=0), b.lens, b.new,
                                                        p_eps=P_EPS[which], **b.scales, **kw)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert ((lse.cpu().double() - want_lse).abs() <= lse_bound).all()


@pytest.mark.parametrize("which", ["step", "chunk"])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.02, 1.5])
def test_scales(ops, dev, which, dtype, cache, scale):
    b = batch(which, dtype, cache)
    call, args = arguments(ops, dev, b, which)
    lse = torch.full(b.query.shape[:2], 77.0, device=dev)
    out = call(*args, scale=scale, lse=lse, check=True, **b.scales)
    check(b, which, out, lse, scale=scale)


@pytest.mark.parametrize("which", ["step", "chunk"])
def test_replays(ops, dev, which):
    b = batch(which, F16, F16, seed=3)
    call, args = arguments(ops, dev, b, which)
    out = torch.zeros(b.query.shape, dtype=F16, device=dev)
    lse = torch.zeros(b.query.shape[:2], device=dev)
    call(*args, out=out, lse=lse, check=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(*args, out=out, lse=lse, check=False)
    for _ in range(3):
        out.fill_(77.0)
        lse.fill_(77.0)
        graph.replay()
        torch.cuda.synchronize()
        ops.check_status(dev)
        check(b, which, out, lse)
