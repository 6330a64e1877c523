"""CPU: attention over 4-bit caches does not look at the head strides of its
descriptor (rows hold all heads)."""
from __future__ import annotations

import ctypes

import pytest

from kv_cache_adapter_b200 import _lib
from test_attend_refusals import desc


@pytest.mark.parametrize("strides", [(0, 0), (8, 256), (256, 8), (1, -3)])
def test_head_strides_are_not_looked_at(strides):
    d = desc(cache_type=_lib.KVCA_TYPE_E2M1, key_head_stride=strides[0], value_head_stride=strides[1], num_seqs=0)
    lib = _lib.load()
    assert lib.kvca_attend_step(ctypes.byref(d), None, 0, None, None, None) == _lib.KVCA_OK
    d.cache_type = _lib.KVCA_TYPE_F16
    aligned = strides[0] % 16 == 0 and strides[1] % 16 == 0
    want = _lib.KVCA_OK if aligned else _lib.KVCA_ERR_BAD_ARGUMENT
    assert lib.kvca_attend_step(ctypes.byref(d), None, 0, None, None, None) == want


@pytest.mark.parametrize("bad", [dict(key=8), dict(key_block_stride=8), dict(value_token_stride=8)],
                         ids=lambda b: ",".join(b))
def test_other_strides_are(bad):
    d = desc(**{"cache_type": _lib.KVCA_TYPE_E2M1, "num_seqs": 0, **bad})
    assert _lib.load().kvca_attend_step(ctypes.byref(d), None, 0, None, None, None) == _lib.KVCA_ERR_BAD_ARGUMENT
