"""attend_chunk with offsets that are not in order: the sequences that they
spoil are reported and left out, the others attend as ever."""
from __future__ import annotations

import pytest
import torch

import attend_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda

    return kv_cache_adapter_cuda


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def attend(ops, dev, b, offsets):
    key, value = b.on(dev)
    out = torch.full(b.query.shape, 77.0, dtype=b.query.dtype, device=dev)
    with pytest.raises(IndexError):
        ops.attend_chunk(b.query.to(dev), torch.tensor(offsets, device=dev), key, value, b.tables.to(dev),
                         torch.tensor(b.lens, device=dev), out=out, check=True)
    want, _, bound, _ = oracle.attention(b.query, b.key, b.value, b.tables.clamp(min=0), b.lens, b.new, p_eps=2.0 ** -11)
    right = ((out.cpu().double() - want).abs() <= bound).flatten(1).all(1)
    same = (out == 77).flatten(1).all(1).cpu()
    return right, same


# the offset between the second and the third sequence is another; which rows are right and which left alone
@pytest.mark.parametrize("offset,right,same", [(5, (0, 10, 45, 50), (10, 45)), (1 << 40, (0, 10, 45, 50), (10, 45)),
                                               (-3, (0, 10, 45, 50), (10, 45)), (48, (0, 10), (48, 50))])
def test_one_wrong_offset(ops, dev, offset, right, same):
    b = oracle.Batch(lens=[40, 60, 50, 30], new=[10, 20, 15, 5], heads=2, group=2, dim=64, block=16,
                     dtype=torch.float16, seed=1)
    good, kept = attend(ops, dev, b, [0, 10, offset, 45, 50])
    for begin, end in zip(right[::2], right[1::2]):
        assert good[begin:end].all()
    assert kept[same[0]:same[1]].all()


def test_many_wrong_offsets(ops, dev):
    """More rows than there are."""
    b = oracle.Batch(lens=[60, 50, 50, 50, 50, 90], new=[40, 0, 0, 0, 0, 10], heads=1, group=40, dim=64, block=16,
                     dtype=torch.float16, seed=2)
    good, _ = attend(ops, dev, b, [0, 40, 0, 40, 0, 40, 50])
    assert good.all()


def test_wrong_offsets_of_many_sequences(ops, dev):
    """Over several rounds of the planning block: sequences 700 to 1,299 repeat the offsets of 100 to 699."""
    n = 2600
    b = oracle.Batch(lens=[9] * n, new=[1] * n, heads=1, group=2, dim=64, block=16, dtype=torch.float16, seed=3)
    offsets = list(range(n + 1))
    offsets[700:1300] = range(100, 700)
    good, kept = attend(ops, dev, b, offsets)
    assert good[:699].all() and good[1300:].all()
    assert kept[700:1299].all()
