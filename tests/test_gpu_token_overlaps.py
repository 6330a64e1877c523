"""append_tokens with queries rotated where they are, beside the keys and values of one
projection in several orders; and what Python says of those that meet."""
from __future__ import annotations

import pytest
import torch

import token_oracle as oracle
from test_gpu_tokens import BF16, F16, dev, ops, places, rows_of  # noqa: F401

pytestmark = pytest.mark.gpu


def beside(order, rows):
    """Query, key and value rows (rows, heads, 64) of one tensor of bf16 values."""
    if order == "side by side":
        x = rows_of((rows, 12, 64), BF16, 3)
        return x, lambda t: (t[:, :8], t[:, 8:10], t[:, 10:])
    if order == "query last":
        x = rows_of((rows, 12, 64), BF16, 4)
        return x, lambda t: (t[:, 4:], t[:, :2], t[:, 2:4])
    if order == "head by head":
        x = rows_of((rows, 4, 3, 64), BF16, 5)
        return x, lambda t: (t[:, :, 0], t[:, :, 1], t[:, :, 2])
    if order == "side by side in each head":
        x = rows_of((rows, 4, 256), BF16, 6)
        return x, lambda t: (t[..., :64], t[..., 64:128], t[..., 192:])
    x = rows_of((12, rows, 64), BF16, 7)  # heads first
    return x, lambda t: (t[:8].transpose(0, 1), t[8:10].transpose(0, 1), t[10:].transpose(0, 1))


@pytest.mark.parametrize("rows", [1, 2, 37])
@pytest.mark.parametrize("order", ["side by side", "query last", "head by head", "side by side in each head",
                                   "heads first"])
def test_queries_in_place_beside_keys_and_values(ops, dev, order, rows):
    x, split = beside(order, rows)
    q, k, v = split(x)
    live = x.to(dev)
    in_place, *others = split(live)
    heads = k.shape[1]
    kc, vc = (torch.zeros((4, 16, heads, 64), dtype=BF16, device=dev) for _ in range(2))
    at, slots = places(rows, 60, rows), torch.arange(rows)
    table = ops.rotary_table(60, 64)
    got = ops.append_tokens(*others, kc, vc, slots.to(dev), positions=at.to(dev), table=table.to(dev), query=in_place,
                            query_out=in_place, check=True)
    assert got is in_place
    for have, rotated in ((got, q), (kc.flatten(0, 1)[:rows], k)):
        want, bound = oracle.rotate(rotated, at, table)
        oracle.check_rows(have.cpu(), want, bound, BF16)
    assert torch.equal(vc.flatten(0, 1)[:rows].cpu(), v)
    after = split(live.cpu())
    assert torch.equal(after[1], k) and torch.equal(after[2], v)


def test_what_meets_is_named(ops, dev):
    x = torch.zeros((5, 12, 64), dtype=F16, device=dev)
    kc, vc = (torch.zeros((4, 16, 2, 64), dtype=F16, device=dev) for _ in range(2))
    at, table = torch.zeros(5, dtype=torch.int64, device=dev), ops.rotary_table(8, 64).to(dev)
    for key, value in ((x[:, 6:8], x[:, 10:]), (x[:, 8:10], x[:, 7:9]), (x[:, 0:2], x[:, 10:]),
                       (x[:, 8:10], x.view(5, 6, 2, 64)[:, 3:5, 1]), (x[:, 9::2][:, :2], x[:, 1:12:10])):
        with pytest.raises(ValueError, match="query_out must not overlap key or value"):
            ops.append_tokens(key, value, kc, vc, at, positions=at, table=table, query=x[:, :8], query_out=x[:, :8])
    rows = torch.zeros((5, 2, 64), dtype=F16, device=dev)
    inside = kc.view(-1).view(torch.int64)
    angles = vc.view(-1).view(torch.float32)[:512].view(8, 64)
    for slots, positions, turns in ((inside[-5:], at, table), (at, inside[16:21], table), (at, at, angles)):
        with pytest.raises(ValueError, match="caches must not overlap slot_mapping"):
            ops.append_tokens(rows, rows, kc, vc, slots, positions=positions, table=turns)
    assert not kc.any() and not vc.any()


def test_keys_of_one_row_for_all(ops, dev):
    x = rows_of((9, 12, 64), BF16, 8)
    live = x.to(dev)
    kc, vc = (torch.zeros((4, 16, 2, 64), dtype=BF16, device=dev) for _ in range(2))
    at, table = places(9, 60, 9), ops.rotary_table(60, 64)
    key = live[3:4, 8:10].expand(9, 2, 64)
    ops.append_tokens(key, live[:, 10:], kc, vc, torch.arange(9, device=dev), positions=at.to(dev),
                      table=table.to(dev), query=live[:, :8], query_out=live[:, :8], check=True)
    for have, rotated in ((live[:, :8], x[:, :8]), (kc.flatten(0, 1)[:9], x[3:4, 8:10].expand(9, 2, 64))):
        want, bound = oracle.rotate(rotated, at, table)
        oracle.check_rows(have.cpu(), want, bound, BF16)
    with pytest.raises(ValueError, match="query_out must not overlap key or value"):
        ops.append_tokens(live[3:4, 7:9].expand(9, 2, 64), live[:, 10:], kc, vc, torch.arange(9, device=dev),
                          positions=at.to(dev), table=table.to(dev), query=live[:, :8], query_out=live[:, :8])
