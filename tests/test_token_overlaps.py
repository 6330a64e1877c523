"""CPU: memory that a call of append_tokens would write while it is read: refused at
the C ABI (no device needed), and the reason found in Python."""
from __future__ import annotations

import ctypes
import itertools
import random

import pytest

from kv_cache_adapter_b200 import _lib
from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops
from test_token_refusals import append_desc

BAD = _lib.KVCA_ERR_BAD_ARGUMENT

# Queries rotated where they are, 8 heads of 256 bytes; keys and values that begin at a later head of theirs, end in
# their first one, lie in another row's, or in between at another distance of rows or heads.
AT = 1 << 20
IN_PLACE = dict(query_out=AT, query_row_stride=4096, query_out_row_stride=4096, key_row_stride=4096,
                value_row_stride=4096, key=AT + 2048, value=AT + 2560)
IN_PLACE_MEETS = [dict(key=AT + 6 * 256), dict(value=AT + 256), dict(value=AT + 7 * 256 + 16),
                  dict(key=AT + 4096 + 6 * 256), dict(key=AT - 256), dict(value=AT + 3 * 4096 - 16),
                  dict(key_head_stride=2048), dict(value_head_stride=4096 - 512 - 256), dict(key_row_stride=2048),
                  dict(value_row_stride=4096 - 512), dict(key_row_stride=0, key=AT + 4096),
                  dict(query_row_stride=6144, query_out_row_stride=6144, query_head_stride=768,
                       query_out_head_stride=768, key=AT + 256, key_row_stride=6144, key_head_stride=768,
                       value=AT + 768 * 5, value_row_stride=6144, value_head_stride=768)]


@pytest.mark.parametrize("bad", IN_PLACE_MEETS, ids=lambda v: ",".join(v))
def test_queries_in_place_over_keys_or_values(bad):
    d = append_desc(**{**IN_PLACE, **bad})
    assert _lib.load().kvca_append_tokens(ctypes.byref(d), None, None) == BAD


def places(address, rows, row, heads, head, unit):
    return {b for r, h in itertools.product(range(rows), range(heads))
            for b in range(address + r * row + h * head, address + r * row + h * head + unit)}


def test_rows_that_meet():
    """Against all their bytes."""
    rng = random.Random(1)
    met = apart = 0
    for _ in range(3000):
        rows, unit = rng.randint(1, 4), rng.choice((2, 4))
        a = (100, rng.choice((0, 8, 16, 24, 40)), rng.randint(1, 3), rng.choice((0, 2, 4, 6, 8, 12)))
        alike = rng.random() < 0.7
        b = (rng.randint(60, 150) & ~1, a[1] if alike else rng.choice((0, 8, 16, 24)), rng.randint(1, 3),
             a[3] if alike else rng.choice((0, 2, 4, 8, 12)))
        truth = bool(places(a[0], rows, *a[1:], unit) & places(b[0], rows, *b[1:], unit))
        got = ops._rows_meet(rows, a, b, unit)
        assert got == truth, (rows, unit, a, b)
        met, apart = met + truth, apart + (not truth)
    assert met > 300 and apart > 300


# The descriptor's slot_mapping and positions (32 bytes each) lie at 4096, its table (51,200 bytes) at 8192; with the
# strides as they are a cache holds 64 KB.
APART = dict(slot_mapping=1 << 26, positions=1 << 27, table=1 << 28)
CACHE_MEETS = [dict(key_cache=4096), dict(value_cache=4096), {**APART, "slot_mapping": (1 << 24) + 65536 - 8},
               {**APART, "slot_mapping": (1 << 25) - 24}, {**APART, "positions": (1 << 24) + 512},
               {**APART, "positions": (1 << 25) + 65536 - 8}, {**APART, "table": (1 << 24) + 65536 - 16},
               {**APART, "table": (1 << 25) - 51200 + 16},
               {**APART, "table": (1 << 25) - 51200 + 16, "cache_type": _lib.KVCA_TYPE_E2M1},
               {**APART, "slot_mapping": (1 << 24) + 7 * 8192 + 15 * 512, "cache_type": _lib.KVCA_TYPE_E4M3}]


@pytest.mark.parametrize("bad", CACHE_MEETS, ids=lambda v: ",".join(v))
def test_caches_over_what_a_call_reads_of_its_tokens(bad):
    assert _lib.load().kvca_append_tokens(ctypes.byref(append_desc(**bad)), None, None) == BAD
