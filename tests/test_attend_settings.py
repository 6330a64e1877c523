"""CPU: the attention calls' process-wide settings."""
from __future__ import annotations

from kv_cache_adapter_b200 import _lib


def test_wait_limit_is_kept():
    lib = _lib.load()
    assert lib.kvca_attend_wait_limit(-1) == 2_000_000_000
    assert lib.kvca_attend_wait_limit(7) == 2_000_000_000
    assert lib.kvca_attend_wait_limit(-5) == 7
    assert lib.kvca_attend_wait_limit(2_000_000_000) == 7
