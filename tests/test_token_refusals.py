"""CPU: what the token operators refuse before any launch, at the C ABI (no
device needed) and in Python; the rotation's table."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from kv_cache_adapter_b200 import _lib
from kv_cache_adapter_b200 import kv_cache_adapter_cuda as ops

BAD = _lib.KVCA_ERR_BAD_ARGUMENT


def with_changes(d, kw):
    for name, x in kw.items():
        setattr(d, name, x)
    return d


def rotate_desc(**kw):
    return with_changes(_lib.RotateDesc(num_rows=4, x=1 << 20, row_stride=2048, head_stride=256, out=1 << 21,
                                        out_row_stride=2048, out_head_stride=256, positions=4096, table=8192,
                                        table_rows=100, heads=8, head_dim=128, rotary_dim=64, type=_lib.KVCA_TYPE_F16),
                        kw)


def append_desc(**kw):
    return with_changes(
        _lib.AppendDesc(num_rows=4, query=1 << 20, query_row_stride=2048, query_head_stride=256, query_out=1 << 21,
                        query_out_row_stride=2048, query_out_head_stride=256, key=1 << 22, key_row_stride=512,
                        key_head_stride=256, value=1 << 23, value_row_stride=512, value_head_stride=256,
                        key_cache=1 << 24, key_block_stride=8192, key_token_stride=512, key_cache_head_stride=256,
                        value_cache=1 << 25, value_block_stride=8192, value_token_stride=512,
                        value_cache_head_stride=256, num_blocks=8, block_size=16, slot_mapping=4096, positions=4096,
                        table=8192, table_rows=100, q_heads=8, kv_heads=2, head_dim=128, rotary_dim=128,
                        type=_lib.KVCA_TYPE_F16, cache_type=_lib.KVCA_TYPE_F16, key_scale=1.0, value_scale=1.0), kw)


def read_desc(**kw):
    return with_changes(_lib.ReadDesc(cache=1 << 20, block_stride=4096, token_stride=256, head_stride=128, num_blocks=8,
                                      block_size=16, slot_mapping=4096, num_rows=4, kv_heads=2, head_dim=128,
                                      cache_type=_lib.KVCA_TYPE_E4M3, type=_lib.KVCA_TYPE_F16, scale=1.0, out=1 << 21),
                        kw)


ROTATE = [dict(num_rows=-1), dict(heads=0), dict(head_dim=12), dict(head_dim=264), dict(rotary_dim=0),
          dict(rotary_dim=63), dict(rotary_dim=130), dict(table_rows=-1), dict(type=_lib.KVCA_TYPE_E4M3), dict(x=8),
          dict(out=4), dict(row_stride=8), dict(out_head_stride=24), dict(table=8), dict(x=0), dict(out=0),
          dict(positions=None), dict(table=None)]
APPEND = [dict(num_rows=-1), dict(kv_heads=0), dict(q_heads=-1), dict(head_dim=12), dict(head_dim=264),
          dict(num_blocks=-1), dict(block_size=0), dict(type=_lib.KVCA_TYPE_F32), dict(type=_lib.KVCA_TYPE_E4M3),
          dict(cache_type=_lib.KVCA_TYPE_BF16), dict(cache_type=9), dict(cache_type=_lib.KVCA_TYPE_E4M3, head_dim=24),
          dict(cache_type=_lib.KVCA_TYPE_E2M1, head_dim=48), dict(rotary_dim=3), dict(rotary_dim=130),
          dict(rotary_dim=0), dict(table_rows=0, table=None, rotary_dim=0), dict(table=None), dict(positions=None),
          dict(key_scale=2.0), dict(value_scale=0.0), dict(cache_type=_lib.KVCA_TYPE_E4M3, key_scale=0.0),
          dict(cache_type=_lib.KVCA_TYPE_E2M1, value_scale=-1.0),
          dict(cache_type=_lib.KVCA_TYPE_E4M3, value_scale=math.inf),
          dict(cache_type=_lib.KVCA_TYPE_E4M3, key_scale=math.nan), dict(key=8), dict(value_row_stride=8),
          dict(key_token_stride=8), dict(value_cache_head_stride=8), dict(query_out=8), dict(table=8), dict(key=0),
          dict(value=0), dict(key_cache=0), dict(value_cache=0), dict(slot_mapping=None), dict(query=0),
          dict(query_out=0)]
READ = [dict(num_rows=-1), dict(kv_heads=0), dict(head_dim=24), dict(head_dim=272), dict(num_blocks=-1),
        dict(block_size=0), dict(type=_lib.KVCA_TYPE_E4M3), dict(cache_type=_lib.KVCA_TYPE_F16),
        dict(cache_type=_lib.KVCA_TYPE_E2M1, head_dim=48), dict(cache=8), dict(token_stride=8), dict(head_stride=8),
        dict(out=8), dict(cache=0), dict(out=0), dict(slot_mapping=None)]


@pytest.mark.parametrize("call,desc,bad", [("kvca_rotate_tokens", rotate_desc, b) for b in ROTATE]
                         + [("kvca_append_tokens", append_desc, b) for b in APPEND]
                         + [("kvca_read_tokens", read_desc, b) for b in READ],
                         ids=lambda v: ",".join(v) if isinstance(v, dict) else None)
def test_c_abi_refuses(call, desc, bad):
    assert getattr(_lib.load(), call)(ctypes.byref(desc(**bad)), None, None) == BAD


# what is written meets itself, or something that is read (byte ranges of the descriptors above)
FUSED = dict(key=(1 << 20) + 2048, value=(1 << 20) + 2560, query_row_stride=1 << 12, key_row_stride=1 << 12,
             value_row_stride=1 << 12)
MERGED = dict(value_cache=(1 << 24) + 512, key_token_stride=1024, value_token_stride=1024, key_block_stride=16384,
              value_block_stride=16384)
ROTATE_MEETS = [dict(out=(1 << 20) + 256), dict(out=1 << 20, out_row_stride=4096), dict(out_head_stride=128),
                dict(out_row_stride=1024), dict(out_head_stride=0), dict(out=8192), dict(out=4096), dict(out=4112),
                dict(row_stride=-2048), dict(out_head_stride=-256)]
APPEND_MEETS = [dict(query_out=(1 << 20) + 256), dict(query_out=1 << 20, query_out_row_stride=4096),
                dict(query_out_head_stride=0), dict(query_out_row_stride=1024), dict(query_out=8192),
                dict(query_out=4096), dict(query_out=1 << 22), dict(query_out=(1 << 23) + 512),
                dict(query_out=(1 << 20) + 2048, query_out_row_stride=1 << 12, **FUSED),
                dict(query_out=1 << 20, query=1 << 20, key=1 << 20), dict(key_cache=1 << 20), dict(key_cache=1 << 21),
                dict(value_cache=1 << 22), dict(value_cache=(1 << 23) + 1536), dict(value_cache=1 << 24),
                dict(value_cache=(1 << 24) + 256), dict(key_token_stride=256), dict(key_block_stride=4096),
                dict(value_block_stride=0), dict(value_cache_head_stride=0), dict(key_row_stride=-512),
                dict(value_block_stride=-8192), dict(value_cache_head_stride=-256),
                {**MERGED, "value_token_stride": 512}, {**MERGED, "value_cache": (1 << 24) + 256},
                dict(cache_type=_lib.KVCA_TYPE_E2M1, value_cache=(1 << 24) + 64)]
READ_MEETS = [dict(out=1 << 20), dict(out=(1 << 20) + 16), dict(out=(1 << 20) - 1024), dict(out=4096),
              dict(token_stride=-256), dict(cache_type=_lib.KVCA_TYPE_E2M1, out=(1 << 20) + 7 * 4096)]


@pytest.mark.parametrize("call,desc,bad", [("kvca_rotate_tokens", rotate_desc, b) for b in ROTATE_MEETS]
                         + [("kvca_append_tokens", append_desc, b) for b in APPEND_MEETS]
                         + [("kvca_read_tokens", read_desc, b) for b in READ_MEETS],
                         ids=lambda v: ",".join(v) if isinstance(v, dict) else None)
def test_c_abi_refuses_overlaps(call, desc, bad):
    assert getattr(_lib.load(), call)(ctypes.byref(desc(**bad)), None, None) == BAD


@pytest.mark.parametrize("call,desc", [("kvca_rotate_tokens", rotate_desc), ("kvca_append_tokens", append_desc),
                                       ("kvca_read_tokens", read_desc)])
def test_c_abi_nothing_to_do_and_size_limits(call, desc):
    fn = getattr(_lib.load(), call)
    assert fn(None, None, None) == BAD
    assert fn(ctypes.byref(desc(num_rows=0)), None, None) == _lib.KVCA_OK
    assert fn(ctypes.byref(desc(num_rows=1 << 25)), None, None) == _lib.KVCA_ERR_SIZE_LIMIT
    if call != "kvca_rotate_tokens":
        assert fn(ctypes.byref(desc(block_size=1 << 31)), None, None) == _lib.KVCA_ERR_SIZE_LIMIT
        assert fn(ctypes.byref(desc(num_blocks=1 << 60, block_size=1 << 20)), None, None) == _lib.KVCA_ERR_SIZE_LIMIT


@pytest.mark.parametrize("bad", [dict(head_dim=48), dict(head_dim=80), dict(key=8), dict(value_token_stride=24),
                                 dict(query_type=_lib.KVCA_TYPE_E2M1), dict(query_type=_lib.KVCA_TYPE_F32)],
                         ids=lambda b: ",".join(b))
def test_attention_over_four_bits_refuses(bad):
    import test_attend_refusals

    d = test_attend_refusals.desc(**{"cache_type": _lib.KVCA_TYPE_E2M1, "head_dim": 64, **bad})
    lib = _lib.load()
    assert lib.kvca_attend_step(ctypes.byref(d), 4096, 1 << 40, 4096, None, None) == BAD
    assert lib.kvca_attend_step_workspace_bytes(ctypes.byref(d)) == -1
    assert lib.kvca_attend_chunk(ctypes.byref(d), 4096, 4, 4096, 1 << 40, None, None) == BAD
    assert lib.kvca_attend_chunk_workspace_bytes(ctypes.byref(d), 4) == -1


def test_rows_of_four_bit_caches():
    assert ops.e2m1_row_bytes(8, 128) == 8 * (64 + 8)
    assert ops.e2m1_row_bytes(1, 128) == 80 and ops.e2m1_row_bytes(1, 32) == 32 and ops.e2m1_row_bytes(3, 256) == 432
    for heads, dim in ((0, 64), (1, 0), (1, 48), (1, 288), (-1, 64)):
        with pytest.raises(ValueError, match="4-bit"):
            ops.e2m1_row_bytes(heads, dim)
    for dim in range(32, 257, 32):  # heads follow from the row's bytes
        for heads in range(1, 70):
            cache = torch.empty((1, 1, ops.e2m1_row_bytes(heads, dim)), dtype=torch.uint8)
            assert ops._e2m1_heads(cache, dim, "cache") == heads
    with pytest.raises(ValueError, match="no heads"):
        ops._e2m1_heads(torch.empty((1, 1, 96), dtype=torch.uint8), 128, "cache")


def test_python_refuses_cpu_tensors():
    x = torch.zeros((2, 1, 64))
    at = torch.zeros(2, dtype=torch.int64)
    table = ops.rotary_table(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotate_tokens(x, at, table)
    with pytest.raises(TypeError, match="x must be"):
        ops.rotate_tokens([1], at, table)
    cache = torch.zeros((2, 4, 80), dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.append_tokens(x.half(), x.half(), cache, cache, at)
    with pytest.raises(TypeError, match="value must be"):
        ops.append_tokens(x.half(), None, cache, cache, at)
    with pytest.raises(ValueError, match="CUDA"):
        ops.read_tokens(cache, at, head_dim=64)


def test_elements_of_results_share_no_memory():
    ops._distinct((10, 10), (4, 40), 4, "x")
    ops._distinct((3, 2), (80, 16), 16, "x")
    ops._distinct((1, 2), (0, 16), 16, "x")
    for sizes, strides in (((2, 3), (0, 16)), ((2, 3), (32, 16)), ((5, 1), (8, 0))):
        with pytest.raises(ValueError, match="share"):
            ops._distinct(sizes, strides, 16, "x")


def test_packed_descriptors():
    for desc in (_lib.RotateDesc, _lib.AppendDesc, _lib.ReadDesc):
        values = [n + 1 for n in range(len(desc._fields_))]
        assert _lib.packer(desc)(*values) == bytes(desc(*values))


def test_table():
    got = ops.rotary_table(1000, 64, base=10000.0)
    assert got.shape == (1000, 64) and got.dtype == torch.float32
    for p in (0, 1, 7, 999):
        for i in (0, 1, 15, 31):
            angle = p * 10000.0 ** (-2 * i / 64)
            assert abs(got[p, i].item() - math.cos(angle)) <= 2.0 ** -24
            assert abs(got[p, 32 + i].item() - math.sin(angle)) <= 2.0 ** -24
    assert ops.rotary_table(0, 8).shape == (0, 8)


def test_table_scalings():
    plain = ops.rotary_table(64, 64, base=10000.0)
    linear = ops.rotary_table(256, 64, base=10000.0, scaling="linear", factor=4.0)
    assert torch.equal(linear[::4], plain)
    ntk = ops.rotary_table(256, 64, base=10000.0, scaling="ntk", factor=4.0)
    assert torch.allclose(ntk[:64, 0], plain[:, 0], atol=1e-6)  # the fastest angle as it was
    slow = 10000.0 ** (-62 / 64) / 4  # the slowest a quarter of it
    assert abs(ntk[200, 63].item() - math.sin(200 * slow)) < 1e-6
    yarn = ops.rotary_table(256, 64, base=10000.0, scaling="yarn", factor=4.0, original_positions=4096)
    size = 0.1 * math.log(4.0) + 1.0
    assert abs(yarn[3, 0].item() - size * math.cos(3.0)) < 1e-6  # 652 turns within 4,096 positions
    assert abs(yarn[200, 63].item() - size * math.sin(200 * slow)) < 1e-6  # 0.09 turns
    assert abs(yarn[0, 5].item() - size) < 1e-6
    plain_size = ops.rotary_table(4, 64, scaling="yarn", factor=4.0, original_positions=4096, magnitude=1.0)
    assert plain_size[0, 0].item() == 1.0
    # between them the angles fall from one to the other
    rate = torch.atan2(yarn[1, 32:], yarn[1, :32]).double()
    ratio = rate / (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64))
    assert (ratio.diff() <= 1e-6).all() and ratio[0] > 1 - 1e-6 and abs(ratio[-1] - 0.25) < 1e-6


@pytest.mark.parametrize("bad", [dict(rotary_dim=7), dict(rotary_dim=0), dict(num_positions=-1), dict(base=1.0),
                                 dict(base=math.inf), dict(scaling="other"), dict(factor=2.0),
                                 dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0),
                                 dict(scaling="yarn", factor=2.0, original_positions=10, beta_slow=40.0)])
def test_table_refuses(bad):
    with pytest.raises(ValueError):
        ops.rotary_table(**{"num_positions": 4, "rotary_dim": 8, **bad})
