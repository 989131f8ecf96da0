"""Calls of the paged-cache operators at the ends of their sizes (CPU: nothing is launched, no pointer is followed)."""
import os

import pytest
import torch

from test_kv_cache import append_args, attn_args, heads, pages, unlaunched          # noqa: F401
from vortex_amd import _lib, attn_step, kv_cache, rotary_append


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


def test_pages_without_a_head(unlaunched):                              # noqa: F811
    none = torch.zeros(5, 0, 16, 64, dtype=torch.bfloat16)
    for call, args in ((attn_step, attn_args()), (rotary_append, append_args())):
        with pytest.raises(ValueError, match="k_pages"):
            call(**{**args, "k_pages": none, "v_pages": none})
