"""record / release of a paged cache on the CPU (the device's part is PagedKVCache.step, which a recorded step calls)."""
import pytest
import torch

from vortex_amd.kv_cache import PagedKVCache


def recorded(tokens=20, counts=(10, 3), pages=8, max_len=64):
    cache = PagedKVCache(1, 1, 8, pages, max_len, page_size=16, device="cpu")
    cache.add(len(counts))
    cache.extend(list(counts))
    cache.record(tokens)
    return cache


def test_steps_are_counted_once():
    cache = recorded()
    for _ in range(3):
        cache.step()
    cache.release(3)
    for steps in (3, 0):                        # a second release: nothing is recorded any more
        with pytest.raises(RuntimeError, match="recorded"):
            cache.release(steps)
    assert cache.lengths() == [13, 6] == cache.lens.tolist()
    assert cache.extend(4).tolist() == [13, 14, 15, 16, 6, 7, 8, 9]         # across a page's end
    assert cache.lengths() == [17, 10] == cache.lens.tolist()


def test_release_refuses_steps_that_cannot_have_run():
    cache = recorded(tokens=5)
    for steps in (-1, 6):
        with pytest.raises(ValueError, match="5 tokens"):
            cache.release(steps)
        assert cache.recorded and cache.lengths() == [10, 3]
    for _ in range(5):
        cache.step()
    cache.release(5)
    assert cache.lengths() == [15, 8] == cache.lens.tolist()
