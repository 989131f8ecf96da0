"""Paged key / value cache of the attention blocks: the tensor-level calls over the C ABI (attn_step, rotary_append,
kv_copy_pages, rotary_turns) and the host side that hands out pages (PagedKVCache).

The reference keeps one [B, max_seqlen, 2, H, head_dim] tensor per attention layer (vortex/model/cache.py:8-28) and offers
a block table in its kernel wrappers (vortex/ops/attn_interface.py).  Here a layer's cache is two tensors of pages
[pages, kv_heads, page_size, head_dim], row b of an int32 table names the pages of sequence b in order, and a batch may
hold sequences of any lengths; sequences share pages until one of them writes (fork).

Like the functions of ops.py these only enqueue on torch's current stream (of the tensors' device) and keep nothing
from one call for the next.
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import HeadRows, KvPages, KvPools, KvSide
from .ops import _need_cuda, _strides

_ACT = {torch.bfloat16: _lib.HYENA_DTYPE_BF16, torch.float16: _lib.HYENA_DTYPE_F16}
_PAGE = {**_ACT, torch.float8_e4m3fn: _lib.HYENA_DTYPE_F8E4M3}


class _on:
    """The stream to enqueue on: the current one of the tensors' device, which is made current for the call."""

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def _same_device(first, *ts):
    for t in ts:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}: all of a call's tensors share one device")


def _int32(t, name, dim):
    if t.dtype != torch.int32 or t.dim() != dim or (t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1):
        raise TypeError(f"{name} must be an int32 tensor of {dim} dimension(s) with contiguous rows, got {tuple(t.shape)} {t.dtype}")


def _side(t, scale, heads, name):
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name} must be [pages, kv_heads, page_size, head_dim] with contiguous head_dim")
    if scale is not None and (scale.dtype != torch.float32 or tuple(scale.shape) != (heads,) or not scale.is_contiguous()):
        raise ValueError(f"the scale of {name} must be a contiguous float32 [{heads}] tensor")
    p, h, s, _ = _strides(t)
    return KvSide(t.data_ptr(), p, h, s, None if scale is None else scale.data_ptr())


def _kv(k_pages, v_pages, table, k_scale, v_scale, act):
    """hyena_kv_pages of one layer's cache for activations of type `act`."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] tensors of one shape, got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if act not in _ACT or k_pages.dtype != v_pages.dtype or k_pages.dtype not in (act, torch.float8_e4m3fn):
        raise TypeError("bfloat16 or float16 activations with pages of the same type or of float8_e4m3fn are required, got "
                        f"{act} with {k_pages.dtype} and {v_pages.dtype}")
    _int32(table, "table", 2)
    n, heads, size, hd = k_pages.shape
    rows, width = table.shape
    return KvPages(_side(k_pages, k_scale, heads, "k_pages"), _side(v_pages, v_scale, heads, "v_pages"), n, size, heads, hd,
                   table.data_ptr(), table.stride(0) if rows > 1 else width, width, rows, _PAGE[k_pages.dtype], 0)


def _head_rows(t, name, shape, dtype):
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if tuple(t.shape) != shape or (shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be {list(shape)} with contiguous head_dim, got {tuple(t.shape)}")
    s = _strides(t)
    return HeadRows(t.data_ptr(), s[0], s[1])


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
    _need_cuda(q, k, v, positions, turns, k_pages, v_pages, table, seq, k_scale, v_scale, q_out, k_out)
    _same_device(q, k, v, positions, turns, k_pages, v_pages, table, seq, k_scale, v_scale, q_out, k_out)
    kv = _kv(k_pages, v_pages, table, k_scale, v_scale, q.dtype)
    if q.dim() != 3 or q.shape[2] != kv.head_dim:
        raise ValueError(f"q must be [T, heads, {kv.head_dim}], got {tuple(q.shape)}")
    T, heads, hd = q.shape
    small = (T, kv.kv_heads, hd)
    _int32(positions, "positions", 1)
    if seq is not None:
        _int32(seq, "seq", 1)
    if positions.shape[0] != T or (seq is not None and seq.shape[0] != T):
        raise ValueError(f"{T} rows need {T} positions (and sequences)")
    if seq is None and (T % kv.sequences if kv.sequences else T):
        raise ValueError(f"{T} rows over {kv.sequences} sequences: give seq")
    if turns.dtype != torch.float64 or turns.dim() != 1 or not turns.is_contiguous() or 2 * turns.shape[0] > hd:
        raise ValueError(f"turns must be a contiguous float64 tensor of at most {hd // 2} pairs")
    qr, kr, vr = _head_rows(q, "q", (T, heads, hd), q.dtype), _head_rows(k, "k", small, q.dtype), _head_rows(v, "v", small, q.dtype)
    zero = q_out is None
    if zero:
        q_out = torch.empty((T, heads, hd), dtype=q.dtype, device=q.device)
    qo = _head_rows(q_out, "q_out", (T, heads, hd), q.dtype)
    ko = None if k_out is None else _head_rows(k_out, "k_out", small, q.dtype)
    ref = ctypes.byref
    with _on(q.device) as stream:
        rc = _lib.lib().hyena_rotary_append(ref(kv), ref(qr), ref(kr), ref(vr), ref(qo), None if ko is None else ref(ko),
                                            positions.data_ptr(), None if seq is None else seq.data_ptr(), turns.data_ptr(),
                                            2 * turns.shape[0], int(interleaved), int(zero), T, heads, _ACT[q.dtype], stream)
    if rc:
        _lib.check(rc, "hyena_rotary_append")
    return q_out


def attn_step(q, k_pages, v_pages, table, lens, *, scale=None, k_scale=None, v_scale=None, out=None):
    """Attention of one new token per sequence over its cached positions 0..lens[b]-1 (hyena_attn_step).

    q [B, heads, hd] bf16 or f16; k_pages, v_pages, scales as in rotary_append (append the token's own key first);
    heads a multiple of the pages' kv_heads; table [B, width], lens [B] int32.  scale: of the scores, default
    hd^-1/2.  Returns out [B, heads, hd] of q's type; a sequence with lens <= 0 gets zeros."""
    _need_cuda(q, k_pages, v_pages, table, lens, k_scale, v_scale, out)
    _same_device(q, k_pages, v_pages, table, lens, k_scale, v_scale, out)
    kv = _kv(k_pages, v_pages, table, k_scale, v_scale, q.dtype)
    if q.dim() != 3 or q.shape[0] != kv.sequences or q.shape[2] != kv.head_dim or q.shape[1] % kv.kv_heads or not q.shape[1]:
        raise ValueError(f"q must be [{kv.sequences}, a multiple of {kv.kv_heads} heads, {kv.head_dim}], got {tuple(q.shape)}")
    _int32(lens, "lens", 1)
    B, heads, hd = q.shape
    if lens.shape[0] != B:
        raise ValueError(f"{B} sequences need {B} lengths, got {lens.shape[0]}")
    qr = _head_rows(q, "q", (B, heads, hd), q.dtype)
    if out is None:
        out = torch.empty((B, heads, hd), dtype=q.dtype, device=q.device)
    elif out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be contiguous and of q's shape and type")
    L = _lib.lib()
    nws = L.hyena_attn_step_ws_bytes(B, heads, kv.kv_heads, hd)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
    with _on(q.device) as stream:
        rc = L.hyena_attn_step(ctypes.byref(kv), ctypes.byref(qr), lens.data_ptr(), hd ** -0.5 if scale is None else scale,
                               out.data_ptr(), None if ws is None else ws.data_ptr(), nws, heads, _ACT[q.dtype], stream)
    if rc:
        _lib.check(rc, "hyena_attn_step")
    return out


def _pools(t, name):
    if t.dim() < 3:
        raise ValueError(f"{name} must be [pools, pages, ...], got {tuple(t.shape)}")
    st, inner = _strides(t), 1
    for i in range(t.dim() - 1, 1, -1):
        if st[i] != inner and t.shape[i] != 1:
            raise ValueError(f"a page of {name} must be contiguous")
        inner *= t.shape[i]
    es = t.element_size()
    return KvPools(t.data_ptr(), st[0] * es, st[1] * es, t.shape[1]), inner * es


def kv_copy_pages(pools, src, dst, *, dst_pools=None):
    """Copies page src[i] to page dst[i] in every pool, in one launch (hyena_kv_copy_pages).

    pools [pools, pages, ...] of any type with contiguous pages (the keys and values of all layers); src, dst int32 [n].
    dst_pools: the pools to copy into, of the same page shape and type (default: pools itself; then no page may be
    both a source and a destination).  No page may be a destination twice; pairs with a page that is not there are left
    out.  Returns the pools written to."""
    out = pools if dst_pools is None else dst_pools
    _need_cuda(pools, src, dst, out)
    _same_device(pools, src, dst, out)
    _int32(src, "src", 1)
    _int32(dst, "dst", 1)
    if src.shape[0] != dst.shape[0]:
        raise ValueError(f"{src.shape[0]} source pages, {dst.shape[0]} destination pages")
    a, size = _pools(pools, "pools")
    b = a
    if dst_pools is not None:
        if out.dtype != pools.dtype or out.dim() != pools.dim() or out.shape[0] != pools.shape[0] or out.shape[2:] != pools.shape[2:]:
            raise ValueError(f"pools {tuple(pools.shape)} {pools.dtype} do not fit dst_pools {tuple(out.shape)} {out.dtype}")
        b, _ = _pools(out, "dst_pools")
    with _on(pools.device) as stream:
        rc = _lib.lib().hyena_kv_copy_pages(ctypes.byref(a), ctypes.byref(b), pools.shape[0], size, src.data_ptr(),
                                            dst.data_ptr(), src.shape[0], stream)
    if rc:
        _lib.check(rc, "hyena_kv_copy_pages")
    return out
