"""Calls of the paged-cache entry points that no launch can hold are refused by name (CPU: the pointers are never followed)."""
import os

import pytest

from test_kv_cache import heads, pages
from vortex_amd import _lib, kv_cache


def test_too_large_for_a_launch():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built in this tree")
    L, P, EINVAL = _lib.lib(), 4096, -1
    pool = kv_cache._POOLS(P, 1 << 50, 1 << 42, 5)
    for rc in (L.hyena_attn_step(pages(rows=1 << 25), heads(), P, 1.0, P, P, 1 << 50, 4, 0, None),
               L.hyena_attn_step(pages(rows=1 << 24), heads(), P, 1.0, P, P, 1 << 50, 4, 0, None),
               L.hyena_rotary_append(pages(), heads(), heads(), heads(), heads(), None, P, P, P, 64, 0, 0, (1 << 31) - 1, 4, 0, None),
               L.hyena_rotary_append(pages(), heads(), heads(), heads(), heads(), None, P, P, P, 62, 1, 0, (1 << 31) - 1, 4, 0, None),
               L.hyena_kv_copy_pages(pool, pool, 1, 1 << 40, P, P, 1, None)):
        assert rc == EINVAL and b"too many" in L.hyena_last_error_string(), (rc, L.hyena_last_error_string())
