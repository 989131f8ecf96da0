"""record / release of a paged cache on the CPU (the device's part is PagedKVCache.step, which a recorded step calls)."""
import pytest

from test_kv_cache import on_cpu                # noqa: F401
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


def test_pages_that_no_step_reached_are_free_again(on_cpu):             # noqa: F811
    cache = recorded(tokens=54, pages=8)                # to the end of both rows: all eight pages
    table, lens = cache.table, cache.lens
    assert cache.free_pages == 0
    for _ in range(7):
        cache.step()
    cache.release(7)                                    # 17 and 10 positions: two pages and one
    assert cache.free_pages == 5 and cache.table is table and cache.lens is lens
    assert (cache.table >= 0).sum(1).tolist() == [2, 1] and cache.lens.tolist() == [17, 10]
    cache.add(1)
    assert cache.extend([0, 0, 50]).tolist()[-50:] == list(range(50))       # four of the five
    assert cache.compact() == 7
    cache.select([0, 1])
    assert cache.free_pages == 5
    cache.record(1)                                     # recorded again, and released before any step
    cache.release(0)
    assert cache.free_pages == 5 and cache.lengths() == [17, 10] == cache.lens.tolist()


def test_pages_reserved_ahead_of_a_recording_stay(on_cpu):              # noqa: F811
    cache = recorded(tokens=0, pages=8)
    cache.release(0)
    cache.reserve([40, 5])                              # 50 positions: four pages; 8: one
    assert cache.free_pages == 3
    cache.record(20)
    assert cache.free_pages == 2
    cache.release(0)
    assert cache.free_pages == 3
    # a fork's recording copies the page that both hold; the copy stays with its row
    cache.select([1, 1])
    cache.record(1)
    pages = [list(p) for p in cache._pages]
    cache.step()
    cache.release(1)
    assert cache._pages == pages and pages[0] != pages[1] and cache.lengths() == [4, 4] and cache.free_pages == 6


def test_what_the_host_cannot_know_is_refused(on_cpu):                  # noqa: F811
    cache = recorded(tokens=5)
    cache.step()
    with pytest.raises(RuntimeError, match="recorded"):
        cache.dense(0)                                  # by the host's lengths it would leave the last position out
    cache.release(1)
    assert cache.dense(0)[0].shape == (2, 1, 11, 8)
    with pytest.raises(RuntimeError, match="record"):
        cache.step()                                    # nothing would tell the host
    assert cache.lens.tolist() == cache.lengths() == [11, 4]
