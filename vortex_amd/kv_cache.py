"""Paged key / value cache of the attention blocks: the tensor-level calls over the C ABI (attn_step, rotary_append,
kv_copy_pages, rotary_turns) and the host side that hands out pages (PagedKVCache).

The reference keeps one [B, max_seqlen, 2, H, head_dim] tensor per attention layer (vortex/model/cache.py:8-28) and offers
a block table in its kernel wrappers (vortex/ops/attn_interface.py).  Here a layer's cache is two tensors of pages
[pages, kv_heads, page_size, head_dim], row b of an int32 table names the pages of sequence b in order, and a batch may
hold sequences of any lengths; sequences share pages until one of them writes (fork).

Like the functions of ops.py these only enqueue on torch's current stream (of the tensors' device) and keep nothing
from one call for the next.
"""
import math
import struct

import torch

from . import _lib

_ACT = {torch.bfloat16: _lib.HYENA_DTYPE_BF16, torch.float16: _lib.HYENA_DTYPE_F16}
_PAGE = {**_ACT, torch.float8_e4m3fn: _lib.HYENA_DTYPE_F8E4M3}

# The argument structures of include/hyena_mi355x.h as packed bytes: built in a quarter of the time ctypes takes for
# nested Structures, which counts where a call's kernels run for a few microseconds.
_KV_PAGES = struct.Struct("@P3qP P3qP 4q P3q 2i").pack
_HEADS = struct.Struct("@P2q").pack
_POOLS = struct.Struct("@P3q").pack


# torch.cuda.current_stream builds a Stream object and current_device checks for initialisation (tensors of the device
# exist here); these return the handle and the index
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _enqueue(name, index, *args):
    """Calls an entry point on the current stream of device `index`, which is made current for the call."""
    fn = getattr(_lib.lib(), name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _device(first, *ts):
    """Index of the one device that all of a call's tensors are on."""
    index = first.get_device()
    if index < 0:
        raise RuntimeError("vortex_amd operators run on the GPU only (got a CPU tensor); there is no CPU fallback")
    for t in ts:
        if t is not None and t.get_device() != index:
            raise (RuntimeError if t.get_device() < 0 else ValueError)(
                f"tensors on {first.device} and {t.device}: all of a call's tensors share one device (GPU only)")
    return index


def _row_stride(t, name, dim):
    """Checks an int32 vector or matrix with contiguous rows; the matrix's row stride."""
    if t.dtype is not torch.int32 or t.dim() != dim:
        raise TypeError(f"{name} must be an int32 tensor of {dim} dimension(s), got {tuple(t.shape)} {t.dtype}")
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have contiguous rows")
    return st[0]


def _scale(t, heads, name):
    if t is None:
        return 0
    if t.dtype is not torch.float32 or tuple(t.shape) != (heads,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{heads}] tensor")
    return t.data_ptr()


def _kv(k_pages, v_pages, table, k_scale, v_scale, act):
    """hyena_kv_pages of one layer's cache for activations of type `act`, and (kv_heads, head_dim, sequences)."""
    shape = k_pages.shape
    if len(shape) != 4 or shape != v_pages.shape or not shape[1]:
        raise ValueError("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] tensors of one shape, got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    dtype = k_pages.dtype
    if act not in _ACT or v_pages.dtype is not dtype or (dtype is not act and dtype is not torch.float8_e4m3fn):
        raise TypeError("bfloat16 or float16 activations with pages of the same type or of float8_e4m3fn are required, got "
                        f"{act} with {dtype} and {v_pages.dtype}")
    n, heads, size, hd = shape
    kp, kh, ks, k1 = k_pages.stride()
    vp, vh, vs, v1 = v_pages.stride()
    if (k1 != 1 or v1 != 1) and hd > 1:
        raise ValueError("pages must have contiguous head_dim")
    row = _row_stride(table, "table", 2)
    rows, width = table.shape
    return _KV_PAGES(k_pages.data_ptr(), kp, kh, ks, _scale(k_scale, heads, "k_scale"),
                     v_pages.data_ptr(), vp, vh, vs, _scale(v_scale, heads, "v_scale"), n, size, heads, hd,
                     table.data_ptr(), row, width, rows, _PAGE[dtype], 0), heads, hd, rows


def _head_rows(t, name, shape, dtype):
    st = t.stride()
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.shape != shape or (st[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name} must be {list(shape)} with contiguous head_dim, got {tuple(t.shape)}")
    return _HEADS(t.data_ptr(), st[0], st[1])


def rotary_turns(rotary_dim, base=10000.0, *, factor=1.0, scaling="linear", original_length=None, slow_turns=1.0,
                 fast_turns=32.0, device=None):
    """Revolutions per position of the rotary_dim / 2 pairs, float64: the table rotary_append turns by.

    Plain rotary embedding is base^(-2i/rotary_dim) / 2 pi (vortex/model/rotary.py:422-423).  For contexts `factor` times
    longer than the model was trained on:
      scaling="linear"   positions divided by the factor (the reference's rotary_emb_scaling_factor, vortex/model/model.py:77-81)
      scaling="base"     the base stretched to base * factor^(d/(d-2)): the fastest pair keeps its angle, the slowest one
                         is interpolated by the whole factor
      scaling="parts"    pairs that turn more than fast_turns times within original_length keep their angle, those below
                         slow_turns are interpolated, those between are mixed linearly in the number of turns
                         (interpolation "by parts"; its attention temperature goes into attn_step's scale)"""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even")
    if not factor > 0 or not base > 0:
        raise ValueError(f"base {base} and factor {factor} must be positive")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling == "base":
        if rotary_dim <= 2:
            raise ValueError("scaling='base' needs more than one pair")
        base, factor = base * factor ** (rotary_dim / (rotary_dim - 2)), 1.0
    turns = float(base) ** (-i / max(rotary_dim, 1)) / (2 * math.pi)
    if scaling == "parts":
        if original_length is None or not fast_turns > slow_turns:
            raise ValueError("scaling='parts' needs original_length and fast_turns > slow_turns")
        keep = ((turns * original_length - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        turns = turns * keep + turns / factor * (1 - keep)
    elif scaling in ("linear", "base"):
        turns = turns / factor
    else:
        raise ValueError(f"unknown scaling {scaling!r}: 'linear', 'base' or 'parts'")
    return turns.to(device) if device is not None else turns


def rotary_append(q, k, v, positions, turns, k_pages, v_pages, table, *, seq=None, interleaved=False, k_scale=None,
                  v_scale=None, q_out=None, k_out=None):
    """Rotates q and k and writes k and v into the pages at the same positions, in one launch (hyena_rotary_append).

    q [T, heads, hd], k and v [T, kv_heads, hd] bf16 or f16 (any row and head stride of a multiple of 8: views of one
    projection do); positions [T] int32, negative for padding rows, of which nothing is written; turns: rotary_turns().
    Row t belongs to row seq[t] of the table (int32), or without seq to row t // (T / rows).  k_pages, v_pages
    [pages, kv_heads, page_size, hd] of the same type, or float8_e4m3fn holding k / k_scale, v / v_scale (float32
    [kv_heads]).  Returns q_out (rotated q; may be q itself; a new tensor if not given, zero in padding rows);
    k_out, if given, receives the rotated k."""
    index = _device(q, k, v, positions, turns, k_pages, v_pages, table, seq, k_scale, v_scale, q_out, k_out)
    dtype, shape = q.dtype, q.shape
    kv, kv_heads, hd, rows = _kv(k_pages, v_pages, table, k_scale, v_scale, dtype)
    if len(shape) != 3 or shape[2] != hd:
        raise ValueError(f"q must be [T, heads, {hd}], got {tuple(shape)}")
    T, heads, _ = shape
    small = (T, kv_heads, hd)
    _row_stride(positions, "positions", 1)
    if seq is not None:
        _row_stride(seq, "seq", 1)
    if positions.shape[0] != T or (seq is not None and seq.shape[0] != T):
        raise ValueError(f"{T} rows need {T} positions (and sequences)")
    if seq is None and (T % rows if rows else T):
        raise ValueError(f"{T} rows over {rows} sequences: give seq")
    pairs = turns.shape[0] if turns.dim() == 1 else hd
    if turns.dtype is not torch.float64 or 2 * pairs > hd or not turns.is_contiguous():
        raise ValueError(f"turns must be a contiguous float64 tensor of at most {hd // 2} pairs")
    zero = q_out is None
    if zero:
        q_out = torch.empty(shape, dtype=dtype, device=q.device)
    args = (kv, _head_rows(q, "q", shape, dtype), _head_rows(k, "k", small, dtype), _head_rows(v, "v", small, dtype),
            _head_rows(q_out, "q_out", shape, dtype), None if k_out is None else _head_rows(k_out, "k_out", small, dtype))
    if T:
        _enqueue("hyena_rotary_append", index, *args, positions.data_ptr(), None if seq is None else seq.data_ptr(),
                 turns.data_ptr(), 2 * pairs, bool(interleaved), zero, T, heads, _ACT[dtype])
    return q_out


def attn_step(q, k_pages, v_pages, table, lens, *, scale=None, k_scale=None, v_scale=None, out=None):
    """Attention of one new token per sequence over its cached positions 0..lens[b]-1 (hyena_attn_step).

    q [B, heads, hd] bf16 or f16; k_pages, v_pages, scales as in rotary_append (append the token's own key first);
    heads a multiple of the pages' kv_heads; table [B, width], lens [B] int32.  scale: of the scores, default
    hd^-1/2.  Returns out [B, heads, hd] of q's type; a sequence with lens <= 0 gets zeros."""
    index = _device(q, k_pages, v_pages, table, lens, k_scale, v_scale, out)
    dtype, shape = q.dtype, q.shape
    kv, kv_heads, hd, rows = _kv(k_pages, v_pages, table, k_scale, v_scale, dtype)
    if len(shape) != 3 or shape[0] != rows or shape[2] != hd or not shape[1] or shape[1] % kv_heads:
        raise ValueError(f"q must be [{rows}, a multiple of {kv_heads} heads, {hd}], got {tuple(shape)}")
    _row_stride(lens, "lens", 1)
    if lens.shape[0] != rows:
        raise ValueError(f"{rows} sequences need {rows} lengths, got {lens.shape[0]}")
    heads = shape[1]
    qr = _head_rows(q, "q", shape, dtype)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
    elif out.dtype is not dtype or out.shape != shape or not out.is_contiguous():
        raise ValueError("out must be contiguous and of q's shape and type")
    if rows:
        nws = _lib.lib().hyena_attn_step_ws_bytes(kv, heads)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
        _enqueue("hyena_attn_step", index, kv, qr, lens.data_ptr(), hd ** -0.5 if scale is None else scale, out.data_ptr(),
                 None if ws is None else ws.data_ptr(), nws, heads, _ACT[dtype])
    return out


def _pools(t, name):
    """hyena_kv_pools of [pools, pages, ...], and the bytes of a page."""
    if t.dim() < 3:
        raise ValueError(f"{name} must be [pools, pages, ...], got {tuple(t.shape)}")
    st, shape, inner = t.stride(), t.shape, 1
    for i in range(len(st) - 1, 1, -1):
        if st[i] != inner and shape[i] != 1:
            raise ValueError(f"a page of {name} must be contiguous")
        inner *= shape[i]
    es = t.element_size()
    return _POOLS(t.data_ptr(), st[0] * es, st[1] * es, shape[1]), inner * es


def kv_copy_pages(pools, src, dst, *, dst_pools=None):
    """Copies page src[i] to page dst[i] in every pool, in one launch (hyena_kv_copy_pages).

    pools [pools, pages, ...] of any type with contiguous pages (the keys and values of all layers); src, dst int32 [n].
    dst_pools: the pools to copy into, of the same page shape and type (default: pools itself; then no page may be
    both a source and a destination).  No page may be a destination twice; pairs with a page that is not there are left
    out.  Returns the pools written to."""
    out = pools if dst_pools is None else dst_pools
    index = _device(pools, src, dst, out)
    _row_stride(src, "src", 1)
    _row_stride(dst, "dst", 1)
    n = src.shape[0]
    if dst.shape[0] != n:
        raise ValueError(f"{n} source pages, {dst.shape[0]} destination pages")
    a, size = _pools(pools, "pools")
    b = a
    if dst_pools is not None:
        if out.dtype != pools.dtype or out.dim() != pools.dim() or out.shape[0] != pools.shape[0] or out.shape[2:] != pools.shape[2:]:
            raise ValueError(f"pools {tuple(pools.shape)} {pools.dtype} do not fit dst_pools {tuple(out.shape)} {out.dtype}")
        b, _ = _pools(out, "dst_pools")
    if n:
        _enqueue("hyena_kv_copy_pages", index, a, b, pools.shape[0], size, src.data_ptr(), dst.data_ptr(), n)
    return out


class PagedKVCache:
    """Keys and values of a batch of sequences over all attention layers, in pages (the role of vortex/model/cache.py:8-28
    for sequences of different lengths that come, fork and go).

    pools [2*layers, pages, kv_heads, page_size, head_dim] is allocated once; pool 2i holds layer i's keys, 2i + 1 its
    values.  A page holds `page_size` positions of one sequence in every layer.  Pages are handed out as sequences
    grow, shared by forked sequences and copied when one of them writes into a page that others still use.  All counting
    is on the host; table [rows, width] and lens [rows] (int32) are its device copies, which the kernels read.

        cache = PagedKVCache(layers=8, kv_heads=32, head_dim=128, num_pages=4096, max_len=32768)
        cache.add(2)                        # two empty sequences
        pos = cache.extend([100, 37])       # room for their prompts; positions [2 * 100] of the padded batch
        ... rotary_append(q, k, v, pos, turns, *cache.layer(i), cache.table) in every layer
        cache.select([0, 0, 0, 1])          # the first one forked into three
        pos = cache.extend(1)               # one more token each: the shared last page is copied for two of them
        ... attn_step(q, *cache.layer(i), cache.table, cache.lens)
    """

    def __init__(self, layers, kv_heads, head_dim, num_pages, max_len, *, page_size=64, dtype=torch.bfloat16, fp8=False,
                 device="cuda"):
        if dtype not in _ACT:
            raise TypeError(f"a cache of {dtype}: bfloat16 and float16 have kernels")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} is not a power of two from 16 to 65536")
        if head_dim % 8 or not 0 < head_dim <= 256:
            raise ValueError(f"head_dim {head_dim} is not a multiple of 8 up to 256")
        if min(layers, kv_heads, num_pages or 0, max_len) < 1:
            raise ValueError("layers, kv_heads, num_pages and max_len must be positive")
        self.page_size, self.max_len, self.dtype, self.fp8 = page_size, max_len, dtype, fp8
        self.width = -(-max_len // page_size)
        self.pools = torch.empty(2 * layers, num_pages, kv_heads, page_size, head_dim,
                                 dtype=torch.float8_e4m3fn if fp8 else dtype, device=device)
        # per layer and side one scale a head, 1 until calibrated (e4m3 pages only)
        self.scales = torch.ones(2 * layers, kv_heads, dtype=torch.float32, device=device) if fp8 else None
        self._free = list(range(num_pages - 1, -1, -1))
        self._refs = [0] * num_pages
        self._pages, self._len = [], []         # per row: its pages in order, the positions it holds
        self.recorded = False                   # a recorded token step uses table and lens: they stay where they are
        self._room, self._ahead = 0, []         # tokens that it was recorded for, pages that the rows had before
        self._set_rows()

    @property
    def rows(self):
        return len(self._len)

    @property
    def free_pages(self):
        return len(self._free)

    def lengths(self):
        """Positions that each row holds, as the host counts them."""
        return list(self._len)

    def layer(self, i):
        """(k_pages, v_pages) of attention layer i."""
        return self.pools[2 * i], self.pools[2 * i + 1]

    def layer_scales(self, i):
        """k_scale and v_scale of layer i as keyword arguments of rotary_append and attn_step."""
        if self.scales is None:
            return {}
        return dict(k_scale=self.scales[2 * i], v_scale=self.scales[2 * i + 1])

    def dense(self, i):
        """Keys and values of layer i as two [rows, kv_heads, max(lengths), head_dim] tensors of the activations' type,
        zero behind a row's end: for attention of many new tokens at once, where reading the pages once into rows is
        cheaper than reading them for every token."""
        self._not_recorded()                    # the host does not know how far a recorded step has gone
        n = max(self._len, default=0)
        w = -(-n // self.page_size)
        at = self.table[:, :w].clamp(min=0).long()
        behind = torch.arange(w * self.page_size, device=self.lens.device) >= self.lens[:, None]
        out = []
        for s, pages in enumerate(self.layer(i)):
            x = pages.view(torch.uint8)[at].view(pages.dtype) if self.fp8 else pages[at]         # [rows, w, heads, size, hd]
            x = x.permute(0, 2, 1, 3, 4).reshape(self.rows, pages.shape[1], w * self.page_size, pages.shape[3])
            if self.fp8:
                x = (x.float() * self.scales[2 * i + s][:, None, None]).to(self.dtype)
            out.append(x.masked_fill(behind[:, None, :, None], 0)[:, :, :n])
        return tuple(out)

    def _set_rows(self):
        dev = self.pools.device
        self.table = torch.empty((self.rows, self.width), dtype=torch.int32, device=dev)
        self.lens = torch.empty(self.rows, dtype=torch.int32, device=dev)
        self._fill()

    def _fill(self):
        """The host's copy of the table from the lists of pages, and the device's from that."""
        self._host = torch.full((self.rows, self.width), -1, dtype=torch.int32)
        for row, pages in zip(self._host, self._pages):
            row[:len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self._upload()

    def _upload(self):
        if self.rows:
            self.table.copy_(self._host)
            self.lens.copy_(torch.tensor(self._len, dtype=torch.int32))

    def _not_recorded(self):
        if self.recorded:
            raise RuntimeError("a recorded token step uses this cache: release it first")

    def add(self, n=1):
        """n more empty sequences behind the others; returns the index of the first."""
        self._not_recorded()
        if n < 0:
            raise ValueError(f"{n} sequences")
        first = self.rows
        self._pages += [[] for _ in range(n)]
        self._len += [0] * n
        self._set_rows()
        return first

    def select(self, rows):
        """Keeps the named rows, in that order: one named several times is forked (its pages are shared), one not named
        is dropped and its pages are free again."""
        self._not_recorded()
        rows = list(rows)
        if any(not 0 <= r < self.rows for r in rows):
            raise ValueError(f"rows {rows} of {self.rows}")
        pages, lens, seen = [], [], set()
        for r in rows:
            mine = list(self._pages[r])
            if r in seen:                       # pages reserved ahead stay with the first
                mine = mine[:-(-self._len[r] // self.page_size)]
            seen.add(r)
            for p in mine:
                self._refs[p] += 1
            pages.append(mine)
            lens.append(self._len[r])
        for old in self._pages:
            self._drop(old)
        self._pages, self._len = pages, lens
        self._set_rows()

    def _drop(self, pages):
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                self._free.append(p)

    def _give(self, counts):
        """Pages for counts[r] more positions of every row, and own copies of shared pages that would be written to.
        Raises, with nothing changed, where they do not fit.  Returns whether the table changed."""
        ps, need, shared = self.page_size, 0, {}
        for r, n in enumerate(counts):
            if n < 0 or self._len[r] + n > self.max_len:
                raise ValueError(f"row {r}: {n} more positions behind {self._len[r]} (at most {self.max_len})")
            need += max(0, -(-(self._len[r] + n) // ps) - len(self._pages[r]))
            if n and self._len[r] % ps:
                p = self._pages[r][self._len[r] // ps]
                if self._refs[p] - shared.get(p, 0) > 1:
                    shared[p] = shared.get(p, 0) + 1
                    need += 1
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} of {len(self._refs)} free")
        src, dst, changed = [], [], False
        for r, n in enumerate(counts):
            mine = self._pages[r]
            if n and self._len[r] % ps:
                at = self._len[r] // ps
                p = mine[at]
                if self._refs[p] > 1:
                    mine[at] = self._host[r, at] = self._take()
                    self._refs[p] -= 1
                    src.append(p)
                    dst.append(mine[at])
                    changed = True
            for _ in range(-(-(self._len[r] + n) // ps) - len(mine)):
                mine.append(self._take())
                self._host[r, len(mine) - 1] = mine[-1]
                changed = True
        if src:
            self._copy(src, dst)
        return changed

    def _take(self):
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _copy(self, src, dst, dst_pools=None):
        both = torch.tensor([src, dst], dtype=torch.int32, device=self.pools.device)
        kv_copy_pages(self.pools, both[0], both[1], dst_pools=dst_pools)

    def reserve(self, n):
        """Hands out the pages of n more positions of every row ahead (an int or one count a row): extend, or a recorded
        token step, then changes the lengths only."""
        self._not_recorded()
        if self._give(self._counts(n)):
            self._upload()

    def _counts(self, n):
        counts = [n] * self.rows if isinstance(n, int) else list(n)
        if len(counts) != self.rows:
            raise ValueError(f"{len(counts)} counts for {self.rows} rows")
        return counts

    def extend(self, n):
        """Makes room for n more positions of every row (an int or one count a row) and counts them as held: the call
        ahead of a step's appends.  Returns the positions [rows * max(n)] int32 of the (padded) batch of new tokens, -1
        where a row has fewer."""
        self._not_recorded()
        counts = self._counts(n)
        most = max(counts, default=0)
        if self._give(counts):
            self._len = [a + b for a, b in zip(self._len, counts)]
            self._upload()
        else:
            self._len = [a + b for a, b in zip(self._len, counts)]
            if isinstance(n, int):
                self.lens.add_(n)
            else:
                self.lens.copy_(torch.tensor(self._len, dtype=torch.int32))
        if isinstance(n, int) and n == 1:
            return self.lens - 1
        step = torch.arange(most, dtype=torch.int32, device=self.lens.device)
        more = self.lens.new_tensor(counts)[:, None]
        pos = self.lens[:, None] - more + step
        return torch.where(step < more, pos, torch.full_like(pos, -1)).reshape(-1)

    def record(self, tokens):
        """For a recorded token step (a HIP graph): hands out the pages of `tokens` more positions of every row and
        leaves table and lens in place until release().  The step itself calls step()."""
        ahead = [len(pages) for pages in self._pages]
        self.reserve(tokens)
        self.recorded, self._room, self._ahead = True, tokens, ahead

    def step(self):
        """extend(1) on the device alone, inside a recorded step: the host learns of it at release()."""
        if not self.recorded:
            raise RuntimeError("step() moves the lengths of a cache under record(): extend(1) counts a token on the host too")
        self.lens.add_(1)
        return self.lens - 1

    def release(self, steps):
        """Ends record(): `steps` recorded steps have run.  Pages that record() handed out and no step has reached are free
        again."""
        if not self.recorded:
            raise RuntimeError("no recorded token step to release: its steps are counted already")
        if not 0 <= steps <= self._room:
            raise ValueError(f"{steps} steps of a recording for {self._room} tokens")
        self.recorded = False
        self._len = [n + steps for n in self._len]
        spare = False
        for pages, n, ahead in zip(self._pages, self._len, self._ahead):
            keep = max(-(-n // self.page_size), ahead)
            spare |= keep < len(pages)
            self._drop(pages[keep:])
            del pages[keep:]
        if spare:
            self._fill()

    def compact(self):
        """Moves the pages in use to the lowest ids (one launch over all layers) and returns how many they are."""
        self._not_recorded()
        live = sorted(p for p in range(len(self._refs)) if self._refs[p])
        n = len(live)
        src = [p for p in live if p >= n]
        dst = [p for p in range(n) if not self._refs[p]]
        if src:
            self._copy(src, dst)                # a page that moves is never where another one goes
            self._rename(dict(zip(src, dst)), len(self._refs))
        return n

    def _rename(self, to, num_pages):
        refs = [0] * num_pages
        for p, c in enumerate(self._refs):
            if c:
                refs[to.get(p, p)] = c
        self._refs = refs
        self._free = [p for p in range(num_pages - 1, -1, -1) if not refs[p]]
        self._pages = [[to.get(p, p) for p in pages] for pages in self._pages]
        self._fill()

    def resize(self, num_pages):
        """Another number of pages: the ones in use are copied to the lowest ids of new pools."""
        self._not_recorded()
        live = sorted(p for p in range(len(self._refs)) if self._refs[p])
        if num_pages < max(1, len(live)):
            raise ValueError(f"{num_pages} pages for {len(live)} in use")
        pools = torch.empty(self.pools.shape[0], num_pages, *self.pools.shape[2:], dtype=self.pools.dtype,
                            device=self.pools.device)
        if live:
            self._copy(live, list(range(len(live))), dst_pools=pools)
        self.pools = pools
        self._rename({p: i for i, p in enumerate(live)}, num_pages)
