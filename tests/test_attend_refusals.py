"""CPU: what the attention calls refuse before any launch, at the C ABI (no
device needed) and in Python (argument checks on meta-like CPU tensors)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kv_cache_adapter_b200 import _lib


def desc(**kw):
    d = _lib.AttendDesc(key=1 << 20, value=1 << 21, key_block_stride=4096, key_token_stride=256, key_head_stride=256,
                        value_block_stride=4096, value_token_stride=256, value_head_stride=256, num_blocks=8,
                        block_size=16, block_tables=4096, table_stride=4, table_width=4, seq_lens=8192, num_seqs=2,
                        q_heads=8, kv_heads=2, head_dim=128, query_type=_lib.KVCA_TYPE_F16,
                        cache_type=_lib.KVCA_TYPE_F16, scale=1.0, key_scale=1.0, value_scale=1.0, window=0, sinks=0,
                        query=1 << 22, query_row_stride=2048, query_head_stride=256, out=1 << 23, lse=None)
    for name, x in kw.items():
        setattr(d, name, x)
    return d


BAD = [dict(num_seqs=-1), dict(num_blocks=-1), dict(block_size=0), dict(table_width=-1), dict(table_stride=-1),
       dict(window=-1), dict(sinks=-1), dict(q_heads=7), dict(kv_heads=0), dict(q_heads=0), dict(head_dim=0),
       dict(head_dim=12), dict(head_dim=264), dict(query_type=_lib.KVCA_TYPE_E4M3), dict(query_type=9),
       dict(cache_type=_lib.KVCA_TYPE_BF16), dict(cache_type=_lib.KVCA_TYPE_E4M3, head_dim=24), dict(key=8),
       dict(value_token_stride=24), dict(key_head_stride=8), dict(query=4), dict(query_row_stride=8), dict(out=2)]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: ",".join(b))
def test_c_abi_refuses(bad):
    lib = _lib.load()
    d = desc(**bad)
    assert lib.kvca_attend_step(ctypes.byref(d), 4096, 1 << 40, 4096, None, None) == _lib.KVCA_ERR_BAD_ARGUMENT
    assert lib.kvca_attend_step_workspace_bytes(ctypes.byref(d)) == -1


@pytest.mark.parametrize("big", [dict(table_width=1 << 27), dict(num_seqs=1 << 29), dict(q_heads=1 << 20)],
                         ids=lambda b: ",".join(b))
def test_c_abi_size_limits(big):
    lib = _lib.load()
    assert lib.kvca_attend_step(ctypes.byref(desc(**big)), 4096, 1 << 40, 4096, None, None) == _lib.KVCA_ERR_SIZE_LIMIT


def test_c_abi_needs_its_pointers():
    lib = _lib.load()
    for missing in ("query", "out", "seq_lens", "key", "value", "block_tables"):
        d = desc(**{missing: 0 if missing in ("query", "out", "key", "value") else None})
        assert lib.kvca_attend_step(ctypes.byref(d), 4096, 1 << 40, 4096, None, None) == _lib.KVCA_ERR_BAD_ARGUMENT
    assert lib.kvca_attend_step(None, 4096, 1 << 40, 4096, None, None) == _lib.KVCA_ERR_BAD_ARGUMENT
    # nothing to do: succeeds without a device
    assert lib.kvca_attend_step(ctypes.byref(desc(num_seqs=0)), None, 0, None, None, None) == _lib.KVCA_OK


def test_python_refuses_cpu_tensors():
    from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    kv = torch.zeros((2, 16, 1, 64), dtype=torch.float16)
    ids = torch.zeros((1, 2), dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attend_step(q, kv, kv, ids, ids[0, :1])
    with pytest.raises(TypeError, match="seq_lens"):
        ops.attend_step(q, kv, kv, ids, [3])
