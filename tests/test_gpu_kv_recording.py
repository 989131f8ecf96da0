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


def test_recording_on_a_pool_smaller_than_every_rows_longest():
    # 2 rows of up to 800 tokens would need 100 pages; 2 * 14 are there
    m, L, n = model(), 200, 16
    ids, ipd, want = started(m, L, n, eager=4, max_seqlen=800, num_pages=2 * 14)
    cache = ipd["mha"].cache
    with pytest.raises(RuntimeError, match="pages needed"):
        RecordedDecodeStep(m, ipd, 2)
    for tokens in (0, -3):
        with pytest.raises(ValueError):
            RecordedDecodeStep(m, ipd, 2, tokens=tokens)
    with pytest.raises(ValueError, match="more positions"):
        RecordedDecodeStep(m, ipd, 2, tokens=700)
    assert not cache.recorded and cache.lengths() == [L + 4] * 2 and cache.free_pages == 2
    rec = RecordedDecodeStep(m, ipd, 2, tokens=6)
    assert cache.free_pages == 0                        # a page each from position 208 on
    for i in range(5, 11):
        advance(ipd, L)
        near(rec(ids[:, L + i - 1:L + i])[:, -1], want[:, i])
    with pytest.raises(RuntimeError, match="6 tokens"):
        rec(ids[:, :1])
    rec.release()
    assert cache.free_pages == 0 and cache.lengths() == [L + 10] * 2 == cache.lens.tolist()
    advance(ipd, L)
    near(m(ids[:, L + 10:L + 11], ipd)[:, -1], want[:, 11])
    rec = RecordedDecodeStep(m, ipd, 2, tokens=4)       # and again
    for i in range(12, n):
        advance(ipd, L)
        near(rec(ids[:, L + i - 1:L + i])[:, -1], want[:, i])
    rec.release()
    assert cache.lengths() == [L + 15] * 2 == cache.lens.tolist()


def test_a_recording_for_some_tokens_on_a_dense_cache():
    m, L = model(), 200
    ids = tokens(2, L + 8, 4)
    ipd = m.initialize_inference_params(L + 8)
    m(ids[:, :L], ipd)
    for i in range(1, 5):
        advance(ipd, L)
        m(ids[:, L + i - 1:L + i], ipd)
    advance(ipd, L)
    rec = RecordedDecodeStep(m, ipd, 2, tokens=1)
    rec(ids[:, L + 4:L + 5])
    with pytest.raises(RuntimeError, match="1 token"):
        rec(ids[:, L + 5:L + 6])


def test_an_eager_token_between_replays_is_refused():
    # it would move the lengths on the device without anybody counting it
    m, L, n = model(pattern=("hcs", "attn"), num_layers=2), 200, 9
    ids, ipd, want = started(m, L, n, eager=4)
    rec = RecordedDecodeStep(m, ipd, 2)
    for i in (5, 6):
        advance(ipd, L)
        near(rec(ids[:, L + i - 1:L + i])[:, -1], want[:, i])
        with pytest.raises(RuntimeError, match="release"):
            m(ids[:, L + i - 1:L + i], ipd)
    rec.release()
    cache = ipd["mha"].cache
    assert cache.lengths() == [L + 6] * 2 == cache.lens.tolist()
    advance(ipd, L)
    near(m(ids[:, L + 6:L + 7], ipd)[:, -1], want[:, 7])
