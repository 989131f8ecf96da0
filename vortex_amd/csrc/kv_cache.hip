// Paged key / value cache: rotary positions with the append, and page copies.
#include "kv_cache.h"

int kv_pages_check(const hyena_kv_pages* kv, int dtype, KvPages* out, const char* who) {
    if (!kv || !kv->k.ptr || !kv->v.ptr || !kv->table)
        return hyena_fail(HYENA_EINVAL, "%s: pages and table are required", who);
    if (dtype != HYENA_DTYPE_BF16 && dtype != HYENA_DTYPE_F16)
        return hyena_fail(HYENA_ENOSUP, "%s: activations of type %d (bfloat16 and float16 have kernels)", who, dtype);
    if (kv->dtype != dtype && kv->dtype != HYENA_DTYPE_F8E4M3)
        return hyena_fail(HYENA_ENOSUP, "%s: pages of type %d with activations of type %d", who, kv->dtype, dtype);
    if (kv->num_pages <= 0 || kv->num_pages >= (1LL << 31) || kv->kv_heads <= 0 || kv->kv_heads > 65535 || kv->sequences < 0 ||
        kv->sequences >= (1LL << 31) || kv->table_width < 0 || kv->table_width >= (1LL << 31) || kv->head_dim <= 0)
        return hyena_fail(HYENA_EINVAL, "%s: bad sizes pages=%lld kv_heads=%lld sequences=%lld table_width=%lld head_dim=%lld", who,
                          (long long)kv->num_pages, (long long)kv->kv_heads, (long long)kv->sequences,
                          (long long)kv->table_width, (long long)kv->head_dim);
    if (kv->head_dim % 8 != 0 || kv->head_dim > 256)
        return hyena_fail(HYENA_ENOSUP, "%s: head_dim %lld is not a multiple of 8 up to 256", who, (long long)kv->head_dim);
    if (kv->page_size < 16 || kv->page_size > 65536 || (kv->page_size & (kv->page_size - 1)) != 0)
        return hyena_fail(HYENA_ENOSUP, "%s: page_size %lld is not a power of two from 16 to 65536", who, (long long)kv->page_size);
    const int64_t es = kv_elem_bytes(kv->dtype);
    const hyena_kv_side* in[2] = {&kv->k, &kv->v};
    KvSide* to[2] = {&out->k, &out->v};
    for (int i = 0; i < 2; ++i) {
        const hyena_kv_side& s = *in[i];
        if (((uintptr_t)s.ptr & 15) || s.page_stride % 8 || s.head_stride % 8 || s.slot_stride % 8)
            return hyena_fail(HYENA_EALIGN, "%s: pages must be 16-byte aligned with strides of a multiple of 8 elements", who);
        *to[i] = {(char*)s.ptr, s.page_stride * es, s.head_stride * es, s.slot_stride * es, s.scale};
    }
    out->table = kv->table;
    out->table_stride = kv->table_stride;
    out->num_pages = (int32_t)kv->num_pages;
    out->kv_heads = (int32_t)kv->kv_heads;
    out->head_dim = (int32_t)kv->head_dim;
    out->page_shift = __builtin_ctzll((unsigned long long)kv->page_size);
    out->sequences = (int32_t)kv->sequences;
    out->reach = kv->table_width << out->page_shift;
    return 0;
}

namespace {

struct Heads {
    char* ptr;
    int64_t token_stride, head_stride;      // bytes
};

struct AppendArgs {
    KvPages kv;
    Heads q, k, v, q_out, k_out;
    const int32_t *pos, *seq;
    const double* turns;
    int32_t heads, half, per_seq;           // half = rotary_dim / 2
    int32_t interleaved, zero_skipped;
};

// One block per token; a thread takes pairs (rotated part) and single elements (the rest) of every head in turn.
template <int DT, int KVDT>
__global__ void __launch_bounds__(256) rotary_append_kernel(AppendArgs a) {
    typedef KvElem<DT> E;
    typedef KvElem<KVDT> P;
    typedef typename E::raw raw;
    typedef typename P::raw praw;
    const int64_t t = blockIdx.x;
    const int64_t pos = a.pos[t];
    const int hd = a.kv.head_dim, K = a.kv.kv_heads, half = a.half;
    if (pos < 0 && !a.zero_skipped) return;
    const int64_t s = a.seq ? a.seq[t] : t / a.per_seq;
    int64_t page = -1;
    if (pos >= 0 && s >= 0 && s < a.kv.sequences && pos < a.kv.reach) {
        page = a.kv.table[s * a.kv.table_stride + (pos >> a.kv.page_shift)];
        if (page >= a.kv.num_pages) page = -1;
    }
    const int64_t slot = pos & ((1LL << a.kv.page_shift) - 1);
    const int units = half + (hd - 2 * half);                // pairs, then single elements
    for (int w = threadIdx.x; w < units * (a.heads + 2 * K); w += 256) {
        const int hh = w / units, u = w % units;
        const bool is_q = hh < a.heads, is_v = hh >= a.heads + K;
        const int h = is_q ? hh : (is_v ? hh - a.heads - K : hh - a.heads);
        const Heads& src = is_q ? a.q : (is_v ? a.v : a.k);
        const raw* x = (const raw*)(src.ptr + t * src.token_stride + h * src.head_stride);
        const bool pair = u < half;
        const int i0 = pair ? (a.interleaved ? 2 * u : u) : half + u, i1 = a.interleaved ? 2 * u + 1 : u + half;
        float y0 = E::get(x[i0]), y1 = pair ? E::get(x[i1]) : 0.f;
        if (pair && !is_v) {
            const double turn = (double)pos * a.turns[u];
            float sn, cs;
            sincospif(2.f * (float)(turn - rint(turn)), &sn, &cs);
            const float x0 = y0, x1 = y1;
            y0 = x0 * cs - x1 * sn;
            y1 = x0 * sn + x1 * cs;
        }
        const Heads& dst = is_q ? a.q_out : a.k_out;
        if (!is_v && dst.ptr && (pos >= 0 || is_q)) {
            raw* y = (raw*)(dst.ptr + t * dst.token_stride + h * dst.head_stride);
            y[i0] = pos < 0 ? 0 : E::put(y0);
            if (pair) y[i1] = pos < 0 ? 0 : E::put(y1);
        }
        if (!is_q && page >= 0) {
            const KvSide& side = is_v ? a.kv.v : a.kv.k;
            praw* y = (praw*)(side.ptr + page * side.page_stride + h * side.head_stride + slot * side.slot_stride);
            const float sc = side.scale ? side.scale[h] : 1.f;
            y[i0] = P::put(y0 / sc);
            if (pair) y[i1] = P::put(y1 / sc);
        }
    }
}

// One block per (pair, pool): the page in 16-byte pieces, then its last bytes.
__global__ void __launch_bounds__(256) copy_pages_kernel(const char* src_base, int64_t src_pool, int64_t src_page, int64_t src_pages,
                                                         char* dst_base, int64_t dst_pool, int64_t dst_page, int64_t dst_pages,
                                                         int64_t bytes, const int32_t* src, const int32_t* dst, int wide) {
    const int64_t s = src[blockIdx.x], d = dst[blockIdx.x];
    if (s < 0 || s >= src_pages || d < 0 || d >= dst_pages) return;
    const char* from = src_base + (int64_t)blockIdx.y * src_pool + s * src_page;
    char* to = dst_base + (int64_t)blockIdx.y * dst_pool + d * dst_page;
    const int64_t n16 = wide ? bytes / 16 : 0;
    for (int64_t i = threadIdx.x; i < n16; i += 256) ((u32x4*)to)[i] = ((const u32x4*)from)[i];
    for (int64_t i = 16 * n16 + threadIdx.x; i < bytes; i += 256) to[i] = from[i];
}

int heads_check(const hyena_heads* h, bool required, const char* name, Heads* out, const char* who) {
    *out = {nullptr, 0, 0};
    if (!h || !h->ptr) return required ? hyena_fail(HYENA_EINVAL, "%s: %s is required", who, name) : 0;
    if (((uintptr_t)h->ptr & 15) || h->token_stride % 8 || h->head_stride % 8)
        return hyena_fail(HYENA_EALIGN, "%s: %s must be 16-byte aligned with strides of a multiple of 8 elements", who, name);
    *out = {(char*)h->ptr, h->token_stride * 2, h->head_stride * 2};
    return 0;
}

}  // namespace

extern "C" int hyena_rotary_append(const hyena_kv_pages* kv, const hyena_heads* q, const hyena_heads* k, const hyena_heads* v,
                                   const hyena_heads* q_out, const hyena_heads* k_out, const int32_t* pos, const int32_t* seq,
                                   const double* turns, int64_t rotary_dim, int interleaved, int zero_skipped,
                                   int64_t tokens, int64_t heads, int dtype, void* stream) {
    const char* who = "hyena_rotary_append";
    AppendArgs a;
    int rc = kv_pages_check(kv, dtype, &a.kv, who);
    if (rc) return rc;
    if ((rc = heads_check(q, true, "q", &a.q, who)) || (rc = heads_check(k, true, "k", &a.k, who)) ||
        (rc = heads_check(v, true, "v", &a.v, who)) || (rc = heads_check(q_out, true, "q_out", &a.q_out, who)) ||
        (rc = heads_check(k_out, false, "k_out", &a.k_out, who)))
        return rc;
    if (!pos || (rotary_dim > 0 && !turns)) return hyena_fail(HYENA_EINVAL, "%s: pos and turns are required", who);
    if (tokens < 0 || tokens >= (1LL << 31) || heads <= 0 || heads > 65535)
        return hyena_fail(HYENA_EINVAL, "%s: bad sizes tokens=%lld heads=%lld", who, (long long)tokens, (long long)heads);
    if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > kv->head_dim)
        return hyena_fail(HYENA_EINVAL, "%s: rotary_dim %lld is not an even number up to head_dim %lld", who,
                          (long long)rotary_dim, (long long)kv->head_dim);
    if (tokens == 0) return 0;
    if (!seq && (kv->sequences == 0 || tokens % kv->sequences))
        return hyena_fail(HYENA_EINVAL, "%s: without seq, tokens (%lld) must be a multiple of the sequences (%lld)", who,
                          (long long)tokens, (long long)kv->sequences);
    a.pos = pos;
    a.seq = seq;
    a.turns = turns;
    a.heads = (int32_t)heads;
    a.half = (int32_t)(rotary_dim / 2);
    a.per_seq = seq ? 1 : (int32_t)(tokens / kv->sequences);
    a.interleaved = interleaved != 0;
    a.zero_skipped = zero_skipped != 0;
    hipStream_t s = (hipStream_t)stream;
#define RA_CASE(D, P)                                                                                       \
    if (dtype == D && kv->dtype == P)                                                                       \
        hipLaunchKernelGGL((rotary_append_kernel<D, P>), dim3((unsigned)tokens), dim3(256), 0, s, a);
    RA_CASE(HYENA_DTYPE_BF16, HYENA_DTYPE_BF16)
    RA_CASE(HYENA_DTYPE_F16, HYENA_DTYPE_F16)
    RA_CASE(HYENA_DTYPE_BF16, HYENA_DTYPE_F8E4M3)
    RA_CASE(HYENA_DTYPE_F16, HYENA_DTYPE_F8E4M3)
#undef RA_CASE
    return hyena_check_launch(who);
}

extern "C" int hyena_kv_copy_pages(const hyena_kv_pools* src_pools, const hyena_kv_pools* dst_pools, int64_t pools,
                                   int64_t page_bytes, const int32_t* src, const int32_t* dst, int64_t copies, void* stream) {
    const char* who = "hyena_kv_copy_pages";
    if (!src_pools || !dst_pools) return hyena_fail(HYENA_EINVAL, "%s: pools are required", who);
    if (pools < 0 || copies < 0 || page_bytes < 0 || src_pools->pages < 0 || dst_pools->pages < 0 || pools > 65535 ||
        copies >= (1LL << 31))
        return hyena_fail(HYENA_EINVAL, "%s: bad sizes pools=%lld copies=%lld page_bytes=%lld", who, (long long)pools,
                          (long long)copies, (long long)page_bytes);
    if (pools == 0 || copies == 0 || page_bytes == 0) return 0;
    if (!src_pools->base || !dst_pools->base || !src || !dst)
        return hyena_fail(HYENA_EINVAL, "%s: pools, src and dst are required", who);
    const int wide = !(((uintptr_t)src_pools->base | (uintptr_t)dst_pools->base | src_pools->pool_stride | dst_pools->pool_stride |
                        src_pools->page_stride | dst_pools->page_stride) & 15);
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)copies, (unsigned)pools), dim3(256), 0, (hipStream_t)stream,
                       (const char*)src_pools->base, src_pools->pool_stride, src_pools->page_stride, src_pools->pages,
                       (char*)dst_pools->base, dst_pools->pool_stride, dst_pools->page_stride, dst_pools->pages, page_bytes,
                       src, dst, wide);
    return hyena_check_launch(who);
}
