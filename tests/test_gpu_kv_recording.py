"""RecordedDecodeStep on a paged cache: what it reserves, what it gives back, and what it refuses."""
import pytest
import torch

from test_gpu_kv_model import model, near, tokens
from vortex_amd.model import RecordedDecodeStep

pytestmark = pytest.mark.gpu


def started(m, L, n, seed=4, eager=2, B=2, **kw):
    """A paged cache behind a prompt of L tokens and `eager` token steps; (ids, its caches, the dense cache's logits)."""
    ids = tokens(B, L + n, seed)
    _, want = m.generate(ids[:, :L], n, forced=ids[:, L:])
    ipd = m.initialize_inference_params(kw.pop("max_seqlen", L + n), kv="paged", rows=B, page_size=16, **kw)
    m(ids[:, :L], ipd)
    for i in range(1, eager + 1):
        advance(ipd, L)
        near(m(ids[:, L + i - 1:L + i], ipd)[:, -1], want[:, i])
    return ids, ipd, want


def advance(ipd, L):
    for p in ipd.values():
        p.seqlen_offset = L if p.seqlen_offset == 0 else p.seqlen_offset + 1


def test_a_refused_recording_leaves_the_callers_alone():
    # the caller has the cache under record() for steps of its own: another recording is refused and changes nothing
    m, L, n = model(), 200, 12
    ids, ipd, want = started(m, L, n, eager=4)
    cache = ipd["mha"].cache
    cache.record(3)
    table, free, lens = cache.table.clone(), cache.free_pages, cache.lengths()
    with pytest.raises(RuntimeError, match="recorded"):
        RecordedDecodeStep(m, ipd, 2)
    assert cache.recorded and cache.lengths() == lens and cache.free_pages == free and torch.equal(cache.table, table)
    cache.release(0)
    advance(ipd, L)
    near(m(ids[:, L + 4:L + 5], ipd)[:, -1], want[:, 5])


def test_released_once_and_for_all():
    m, L, n = model(), 200, 12
    ids, ipd, want = started(m, L, n, eager=4)
    rec = RecordedDecodeStep(m, ipd, 2)
    for i in (5, 6, 7):
        advance(ipd, L)
        near(rec(ids[:, L + i - 1:L + i])[:, -1], want[:, i])
    rec.release()
    again = RecordedDecodeStep(m, ipd, 2)
    rec.release()                               # a second time, while another one is in use
    with pytest.raises(RuntimeError, match="released"):
        rec(ids[:, :1])
    assert ipd["mha"].cache.recorded
    advance(ipd, L)
    near(again(ids[:, L + 7:L + 8])[:, -1], want[:, 8])
    again.release()
    again.release()
    cache = ipd["mha"].cache
    assert cache.lengths() == [L + 8] * 2 == cache.lens.tolist()
    for i in range(9, n):
        advance(ipd, L)
        near(m(ids[:, L + i - 1:L + i], ipd)[:, -1], want[:, i])
    assert cache.lengths() == cache.lens.tolist()


def test_a_released_step_on_a_dense_cache_is_refused():
    m, L = model(), 200
    ids = tokens(2, L + 8, 4)
    ipd = m.initialize_inference_params(L + 8)
    m(ids[:, :L], ipd)
    for i in range(1, 5):
        advance(ipd, L)
        m(ids[:, L + i - 1:L + i], ipd)
    advance(ipd, L)
    rec = RecordedDecodeStep(m, ipd, 2)
    rec(ids[:, L + 4:L + 5])
    rec.release()
    rec.release()
    with pytest.raises(RuntimeError, match="released"):
        rec(ids[:, :1])
