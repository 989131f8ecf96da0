"""Paged cache on the CPU: the page accounting of PagedKVCache against a plain model of the sequences' contents, and every
refusal of the operators (before anything is enqueued)."""
import os
import random

import pytest
import torch

from vortex_amd import _lib, kv_cache
from vortex_amd.kv_cache import PagedKVCache, attn_step, kv_copy_pages, rotary_append

BF, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture
def on_cpu(monkeypatch):
    """kv_copy_pages on CPU tensors, by its definition (sources are read before any destination is written)."""
    def copy(pools, src, dst, *, dst_pools=None):
        out = pools if dst_pools is None else dst_pools
        s, d = src.tolist(), dst.tolist()
        assert len(set(d)) == len(d) and (dst_pools is not None or not set(s) & set(d))
        out[:, d] = pools[:, s].clone()
        return out

    monkeypatch.setattr(kv_cache, "kv_copy_pages", copy)


def write(cache, pos, values):
    """The append, on the CPU: value t at position pos[t] of row t // (T / rows), in every pool."""
    per = len(pos) // cache.rows
    for t, p in enumerate(pos):
        if p >= 0:
            cache.pools[:, cache.table[t // per, p // cache.page_size], :, p % cache.page_size] = float(values[t])


def contents(cache, row):
    return [float(cache.pools[0, cache.table[row, p // cache.page_size], 0, p % cache.page_size, 0])
            for p in range(int(cache.lens[row]))]


def check(cache, want):
    assert cache.lens.tolist() == [len(w) for w in want] == cache.lengths()
    for r, w in enumerate(want):
        assert contents(cache, r) == w
        for pool in range(cache.pools.shape[0]):        # every pool moved the same way
            for p in range(0, len(w), 7):
                assert float(cache.pools[pool, cache.table[r, p // cache.page_size], 0, p % cache.page_size, 0]) == w[p]
    used = {p for pages in cache._pages for p in pages}
    assert sorted(used | set(cache._free)) == list(range(len(cache._refs))) and not used & set(cache._free)
    assert all(cache._refs[p] == sum(p in pages for pages in cache._pages) for p in range(len(cache._refs)))


@pytest.mark.parametrize("seed", range(6))
def test_random_lives_of_sequences(on_cpu, seed):
    r = random.Random(seed)
    cache = PagedKVCache(2, 1, 8, 60, 200, page_size=16, device="cpu")
    want, stamp = [], 0
    for _ in range(60):
        op = r.choice(["add", "extend", "extend", "extend", "select", "compact", "resize", "reserve"])
        if op == "add" and cache.rows < 6:
            cache.add(1)
            want.append([])
        elif op == "extend" and cache.rows:
            n = r.choice([1, 1, r.randint(0, 40)])
            counts = n if r.random() < 0.5 else [r.randint(0, n) for _ in want]
            ns = [counts] * len(want) if isinstance(counts, int) else counts
            before = [list(w) for w in want]
            try:
                pos = cache.extend(counts).tolist()
            except (RuntimeError, ValueError):
                check(cache, before)                    # refused with nothing changed
                continue
            most = max(ns)
            assert len(pos) == most * len(want)
            values = []
            for row, n in enumerate(ns):
                assert pos[row * most: row * most + n] == list(range(len(want[row]), len(want[row]) + n))
                assert all(p == -1 for p in pos[row * most + n: (row + 1) * most])
                new = [float((stamp + k) % 251) for k in range(n)]
                stamp += n
                want[row] = want[row] + new
                values += new + [0.0] * (most - n)
            write(cache, pos, values)
        elif op == "select" and cache.rows:
            rows = [r.randrange(cache.rows) for _ in range(r.randint(0, 6))]
            cache.select(rows)
            want = [list(want[i]) for i in rows]
        elif op == "compact":
            n = cache.compact()
            assert all(p < n for pages in cache._pages for p in pages)
        elif op == "reserve" and cache.rows:
            try:
                cache.reserve(r.randint(0, 30))
            except (RuntimeError, ValueError):
                pass
        elif op == "resize":
            live = sum(c > 0 for c in cache._refs)
            cache.resize(max(live + r.randint(0, 30), 30))
        check(cache, want)


def test_forks_share_until_they_write(on_cpu):
    cache = PagedKVCache(1, 1, 8, 8, 100, page_size=16, device="cpu")
    cache.add(1)
    write(cache, cache.extend(40).tolist(), range(40))
    assert cache.free_pages == 5
    cache.select([0, 0, 0])
    assert cache.free_pages == 5                        # nothing copied yet
    write(cache, cache.extend(1).tolist(), [100, 101, 102])
    assert cache.free_pages == 3                        # the last page of two of the three
    check(cache, [[float(x) for x in range(40)] + [100.0 + i] for i in range(3)])
    cache.select([2])
    check(cache, [[float(x) for x in range(40)] + [102.0]])
    assert cache.free_pages == 5
    with pytest.raises(RuntimeError, match="free"):
        cache.add(2) and cache.extend([0, 50, 50])
    with pytest.raises(ValueError):
        cache.extend([70, 0, 0])
    with pytest.raises(ValueError):
        cache.select([3])
    with pytest.raises(ValueError):
        cache.extend([1])
    with pytest.raises(ValueError):
        cache.resize(2)


def test_recorded_steps_count(on_cpu):
    cache = PagedKVCache(1, 1, 8, 8, 40, page_size=16, device="cpu")
    cache.add(2)
    cache.extend([10, 3])
    table = cache.table
    cache.record(30)
    for call in (lambda: cache.add(1), lambda: cache.select([0]), lambda: cache.extend(1), cache.compact, lambda: cache.resize(9)):
        with pytest.raises(RuntimeError, match="recorded"):
            call()
    assert [cache.step().tolist() for _ in range(2)] == [[10, 3], [11, 4]]
    cache.release(2)
    assert cache.lengths() == [12, 5] == cache.lens.tolist() and cache.table is table
    assert cache.extend(1).tolist() == [12, 5]


def test_cache_refusals():
    for bad in (dict(page_size=24), dict(page_size=8), dict(dtype=torch.float32)):
        with pytest.raises((ValueError, TypeError)):
            PagedKVCache(1, 1, 8, 4, 64, device="cpu", **bad)
    for args in ((1, 1, 12, 4, 64), (1, 1, 264, 4, 64), (0, 1, 8, 4, 64), (1, 1, 8, 0, 64)):
        with pytest.raises(ValueError):
            PagedKVCache(*args, device="cpu")


# ---- refusals of the operators: python checks with the device check and the call out of the way ------------------------


@pytest.fixture
def unlaunched(monkeypatch):
    monkeypatch.setattr(kv_cache, "_device", lambda *t: 0)

    def enqueue(name, *a):
        raise AssertionError(f"{name} would have been enqueued")

    monkeypatch.setattr(kv_cache, "_enqueue", enqueue)
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built in this tree")


def attn_args(B=2, H=4, K=2, hd=64, ps=16, W=3, t=BF, pt=None):
    P = 5
    return dict(q=torch.zeros(B, H, hd, dtype=t), k_pages=torch.zeros(P, K, ps, hd, dtype=pt or t),
                v_pages=torch.zeros(P, K, ps, hd, dtype=pt or t), table=torch.zeros(B, W, dtype=torch.int32),
                lens=torch.zeros(B, dtype=torch.int32))


def test_attention_refusals(unlaunched):
    with pytest.raises(AssertionError, match="enqueued"):
        attn_step(**attn_args())
    i32, f32 = torch.int32, torch.float32
    bad = [dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(2, 3, 64, dtype=BF)), dict(q=torch.zeros(3, 4, 64, dtype=BF)),
           dict(q=torch.zeros(2, 4, 32, dtype=BF)), dict(q=torch.zeros(2, 64, 4, dtype=BF).transpose(1, 2)),
           dict(q=torch.zeros(2, 256, dtype=BF)), dict(q=torch.zeros(2, 0, 64, dtype=BF)),
           dict(k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16)), dict(v_pages=torch.zeros(5, 2, 16, 64, dtype=FP8)),
           dict(v_pages=torch.zeros(5, 2, 32, 64, dtype=BF)), dict(k_pages=torch.zeros(5, 2, 16 * 64, dtype=BF)),
           dict(k_pages=torch.zeros(5, 2, 64, 16, dtype=BF).transpose(2, 3)),
           dict(table=torch.zeros(2, 3, dtype=torch.int64)), dict(table=torch.zeros(6, dtype=i32)),
           dict(table=torch.zeros(3, 2, dtype=i32).t()), dict(lens=torch.zeros(3, dtype=i32)),
           dict(lens=torch.zeros(2, dtype=torch.int64)), dict(lens=torch.zeros(4, dtype=i32)[::2]),
           dict(out=torch.zeros(2, 4, 64)), dict(out=torch.zeros(2, 64, 4, dtype=BF).transpose(1, 2)),
           dict(k_scale=torch.zeros(2, dtype=BF)), dict(v_scale=torch.zeros(3, dtype=f32)),
           dict(k_scale=torch.zeros(4, dtype=f32)[::2])]
    for b in bad:
        with pytest.raises((ValueError, TypeError)):
            attn_step(**{**attn_args(), **b})
    with pytest.raises(TypeError):
        attn_step(**attn_args(t=torch.float32))
    empty = attn_args(B=0)
    assert attn_step(**empty).shape == (0, 4, 64)       # no sequence: nothing to enqueue


def append_args(T=4, H=4, K=2, hd=64, ps=16, t=BF, pt=None):
    a = attn_args(2, H, K, hd, ps, 3, t, pt)
    return dict(q=torch.zeros(T, H, hd, dtype=t), k=torch.zeros(T, K, hd, dtype=t), v=torch.zeros(T, K, hd, dtype=t),
                positions=torch.zeros(T, dtype=torch.int32), turns=torch.zeros(hd // 2, dtype=torch.float64),
                k_pages=a["k_pages"], v_pages=a["v_pages"], table=a["table"])


def test_append_refusals(unlaunched):
    with pytest.raises(AssertionError, match="enqueued"):
        rotary_append(**append_args())
    i32 = torch.int32
    bad = [dict(q=torch.zeros(4, 4, 32, dtype=BF)), dict(q=torch.zeros(3, 4, 64, dtype=BF)), dict(k=torch.zeros(4, 4, 64, dtype=BF)),
           dict(v=torch.zeros(4, 2, 64)), dict(k=torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)), dict(q=torch.zeros(4, 256, dtype=BF)),
           dict(positions=torch.zeros(4, dtype=torch.int64)), dict(positions=torch.zeros(5, dtype=i32)),
           dict(turns=torch.zeros(32)), dict(turns=torch.zeros(33, dtype=torch.float64)),
           dict(turns=torch.zeros(32, 1, dtype=torch.float64)), dict(turns=torch.zeros(64, dtype=torch.float64)[::2]),
           dict(seq=torch.zeros(3, dtype=i32)), dict(seq=torch.zeros(4, dtype=torch.int64)),
           dict(table=torch.zeros(3, 3, dtype=i32)),            # four rows over three sequences, no seq
           dict(q_out=torch.zeros(4, 4, 64)), dict(q_out=torch.zeros(4, 2, 64, dtype=BF)), dict(k_out=torch.zeros(4, 4, 64, dtype=BF))]
    for b in bad:
        with pytest.raises((ValueError, TypeError)):
            rotary_append(**{**append_args(), **b})
    none = append_args(T=0)
    assert rotary_append(**none).shape == (0, 4, 64)


def test_copy_refusals(unlaunched):
    i32 = torch.int32
    ok = dict(pools=torch.zeros(2, 6, 3, 16), src=torch.zeros(2, dtype=i32), dst=torch.ones(2, dtype=i32))
    with pytest.raises(AssertionError, match="enqueued"):
        kv_copy_pages(**ok)
    for b in (dict(pools=torch.zeros(2, 6)), dict(pools=torch.zeros(2, 6, 16, 3).transpose(2, 3)), dict(src=torch.zeros(3, dtype=i32)),
              dict(dst=torch.zeros(2, dtype=torch.int64)), dict(dst_pools=torch.zeros(3, 6, 3, 16)),
              dict(dst_pools=torch.zeros(2, 6, 3, 16, dtype=BF)), dict(dst_pools=torch.zeros(2, 9, 3, 8))):
        with pytest.raises((ValueError, TypeError)):
            kv_copy_pages(**{**ok, **b})
    none = torch.zeros(0, dtype=i32)
    assert kv_copy_pages(ok["pools"], none, none) is ok["pools"]


def test_cpu_tensors_are_refused():
    for call in (lambda: attn_step(**attn_args()), lambda: rotary_append(**append_args()),
                 lambda: kv_copy_pages(torch.zeros(2, 6, 3), torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


# ---- refusals at the C entry points: the pointers are never followed -----------------------------------------------------


def pages(ptr=4096, strides=(4096, 1024, 64), n=5, ps=16, K=2, hd=64, table=4096, width=3, rows=2, dtype=0, scale=0):
    return kv_cache._KV_PAGES(ptr, *strides, scale, ptr, *strides, scale, n, ps, K, hd, table, width, width, rows, dtype, 0)


def heads(ptr=4096, tok=256, head=64):
    return kv_cache._HEADS(ptr, tok, head)


def test_c_entry_points_refuse_before_launching():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built in this tree")
    L, P = _lib.lib(), 4096
    EINVAL, EALIGN, ENOSUP = -1, -2, -3
    attn = lambda kv, q=heads(), lens=P, out=P, ws=P, nws=1 << 40, H=4, dt=0: L.hyena_attn_step(kv, q, lens, 1.0, out, ws, nws, H, dt, None)
    wide = dict(width=1 << 20)                          # rows too long for the one-launch form: the workspace counts
    for want, rc in [(EINVAL, attn(None)), (EINVAL, attn(pages(ptr=0))), (EINVAL, attn(pages(table=0))), (ENOSUP, attn(pages(), dt=2)),
                     (ENOSUP, attn(pages(dtype=1))), (ENOSUP, attn(pages(dtype=2))), (EINVAL, attn(pages(n=0))),
                     (EINVAL, attn(pages(K=0))), (EINVAL, attn(pages(hd=0))), (ENOSUP, attn(pages(hd=60))), (ENOSUP, attn(pages(hd=264))),
                     (ENOSUP, attn(pages(ps=8))), (ENOSUP, attn(pages(ps=48))), (ENOSUP, attn(pages(ps=1 << 17))),
                     (ENOSUP, attn(pages(ps=65536, width=1 << 15))), (EALIGN, attn(pages(ptr=4104))),
                     (EALIGN, attn(pages(strides=(4096, 1024, 60)))), (EALIGN, attn(pages(strides=(4092, 1024, 64)))),
                     (EINVAL, attn(pages(), H=3)), (EINVAL, attn(pages(), H=0)), (EINVAL, attn(pages(), q=None)),
                     (EINVAL, attn(pages(), q=heads(0))), (EINVAL, attn(pages(), lens=None)), (EINVAL, attn(pages(), out=None)),
                     (EALIGN, attn(pages(), out=4100)), (EALIGN, attn(pages(), q=heads(4100))), (EALIGN, attn(pages(), q=heads(tok=100))),
                     (EINVAL, attn(pages(**wide), nws=16)), (EINVAL, attn(pages(**wide), ws=None)), (EINVAL, attn(pages(**wide), ws=4100)),
                     (EINVAL, attn(pages(rows=1 << 30), H=4)), (ENOSUP, attn(pages(strides=(1 << 40, 1 << 34, 1 << 28)))),
                     (0, attn(pages(rows=0)))]:
        assert rc == want, L.hyena_last_error_string()
    assert L.hyena_attn_step_ws_bytes(pages(), 4) == 0 < L.hyena_attn_step_ws_bytes(pages(**wide), 4)

    def app(kv=pages(), q=heads(), k=heads(), v=heads(), qo=heads(), ko=None, pos=P, seq=None, turns=P, rd=64, T=4, H=4, dt=0):
        return L.hyena_rotary_append(kv, q, k, v, qo, ko, pos, seq, turns, rd, 0, 0, T, H, dt, None)

    for want, rc in [(EINVAL, app(kv=None)), (EINVAL, app(q=None)), (EINVAL, app(k=None)), (EINVAL, app(v=heads(0))),
                     (EINVAL, app(qo=None)), (EINVAL, app(pos=None)), (EINVAL, app(turns=None)), (EINVAL, app(rd=63)),
                     (EINVAL, app(rd=66)), (EINVAL, app(rd=-2)), (EINVAL, app(T=-1)), (EINVAL, app(T=5)), (EINVAL, app(H=0)),
                     (ENOSUP, app(H=40000)), (EALIGN, app(q=heads(4104))), (EALIGN, app(ko=heads(head=12))), (ENOSUP, app(dt=2)),
                     (EINVAL, app(qo=heads(tok=0))), (EINVAL, app(ko=heads(head=0))), (EINVAL, app(kv=pages(strides=(0, 1024, 64)))),
                     (EINVAL, app(kv=pages(strides=(4096, 0, 64)))), (EINVAL, app(kv=pages(strides=(4096, 1024, 0)))),
                     (ENOSUP, app(q=heads(tok=1 << 28))), (ENOSUP, app(k=heads(head=-64))), (0, app(T=0))]:
        assert rc == want, L.hyena_last_error_string()
    pool = lambda base=P, ps=4096, n=5: kv_cache._POOLS(base, 1 << 20, ps, n)
    copy = lambda a=pool(), b=pool(), n=2, size=64, s=P, d=P, c=3: L.hyena_kv_copy_pages(a, b, n, size, s, d, c, None)
    for want, rc in [(EINVAL, copy(a=None)), (EINVAL, copy(b=pool(base=0))), (EINVAL, copy(s=None)), (EINVAL, copy(n=-1)),
                     (EINVAL, copy(n=70000)), (EINVAL, copy(c=-1)), (EINVAL, copy(c=1 << 31)), (EINVAL, copy(size=-4)),
                     (EINVAL, copy(c=1 << 30, size=1 << 20)), (EINVAL, copy(b=pool(ps=0))), (0, copy(c=0)), (0, copy(n=0)), (0, copy(size=0))]:
        assert rc == want, L.hyena_last_error_string()
