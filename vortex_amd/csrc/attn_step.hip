// Attention of one new token per sequence over a paged key / value cache.
#include "kv_cache.h"

namespace {

struct AttnArgs {
    KvPages kv;
    const char* q;
    int64_t q_seq_stride, q_head_stride;    // bytes
    const int32_t* lens;
    char* out;
    float scale;                            // includes log2(e): the softmax works in powers of two
    int32_t heads, group;
};

// One block per (sequence, head): 256 positions at a time, one score per thread, running maximum and sum.
template <int DT, int KVDT>
__global__ void __launch_bounds__(256) attn_step_kernel(AttnArgs a) {
    typedef KvElem<DT> E;
    typedef KvElem<KVDT> P;
    typedef typename E::raw raw;
    typedef typename P::raw praw;
    __shared__ float q[256], p[256], red[256];
    __shared__ const praw* vrow[256];
    const int h = blockIdx.x % a.heads, b = blockIdx.x / a.heads, kh = h / a.group, tid = threadIdx.x, hd = a.kv.head_dim;
    const int64_t n = min((int64_t)a.lens[b], a.kv.reach);
    const int32_t* table = a.kv.table + b * a.kv.table_stride;
    const float ks = a.scale * (a.kv.k.scale ? a.kv.k.scale[kh] : 1.f);
    if (tid < hd) q[tid] = E::get(((const raw*)(a.q + b * a.q_seq_stride + h * a.q_head_stride))[tid]);
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int64_t j0 = 0; j0 < n; j0 += 256) {
        __syncthreads();
        const int64_t j = j0 + tid;
        float s = -INFINITY;
        vrow[tid] = nullptr;
        if (j < n) {
            const int64_t page = table[j >> a.kv.page_shift], slot = j & ((1LL << a.kv.page_shift) - 1);
            if (page >= 0 && page < a.kv.num_pages) {
                const praw* k = (const praw*)(a.kv.k.ptr + page * a.kv.k.page_stride + kh * a.kv.k.head_stride + slot * a.kv.k.slot_stride);
                vrow[tid] = (const praw*)(a.kv.v.ptr + page * a.kv.v.page_stride + kh * a.kv.v.head_stride + slot * a.kv.v.slot_stride);
                float dot = 0.f;
                for (int d = 0; d < hd; ++d) dot = fmaf(q[d], P::get(k[d]), dot);
                s = dot * ks;
            }
        }
        red[tid] = s;
        __syncthreads();
        for (int w = 128; w > 0; w >>= 1) {
            if (tid < w) red[tid] = (red[tid] >= red[tid + w] || red[tid + w] != red[tid + w]) ? red[tid] : red[tid + w];
            __syncthreads();
        }
        const float mn = fmaxf(m, red[0]), base = mn == -INFINITY ? 0.f : mn;
        p[tid] = vrow[tid] ? exp2f(s - base) : 0.f;
        const float f = exp2f(m - base);
        m = mn;
        l *= f;
        acc *= f;
        __syncthreads();
        for (int i = 0; i < 256; ++i) {
            if (!vrow[i]) continue;
            l += p[i];
            if (tid < hd) acc = fmaf(p[i], P::get(vrow[i][tid]), acc);
        }
    }
    if (tid < hd) {
        const float vs = a.kv.v.scale ? a.kv.v.scale[kh] : 1.f;
        ((raw*)a.out)[((int64_t)b * a.heads + h) * hd + tid] = E::put(l != 0.f ? acc / l * vs : 0.f);
    }
}

}  // namespace

extern "C" int64_t hyena_attn_step_ws_bytes(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim) {
    (void)sequences, (void)heads, (void)kv_heads, (void)head_dim;
    return 0;
}

extern "C" int hyena_attn_step(const hyena_kv_pages* kv, const hyena_heads* q, const int32_t* lens, float scale, void* out,
                               void* ws, int64_t ws_bytes, int64_t heads, int dtype, void* stream) {
    const char* who = "hyena_attn_step";
    AttnArgs a;
    int rc = kv_pages_check(kv, dtype, &a.kv, who);
    if (rc) return rc;
    if (heads <= 0 || heads > 65535 || heads % kv->kv_heads)
        return hyena_fail(HYENA_EINVAL, "%s: %lld heads over %lld key heads", who, (long long)heads, (long long)kv->kv_heads);
    if (kv->sequences == 0) return 0;
    if (!q || !q->ptr || !lens || !out) return hyena_fail(HYENA_EINVAL, "%s: q, lens and out are required", who);
    if (((uintptr_t)q->ptr & 15) || ((uintptr_t)out & 15) || q->token_stride % 8 || q->head_stride % 8)
        return hyena_fail(HYENA_EALIGN, "%s: q and out must be 16-byte aligned with strides of a multiple of 8 elements", who);
    if (kv->sequences * heads >= (1LL << 31))
        return hyena_fail(HYENA_EINVAL, "%s: %lld sequences of %lld heads", who, (long long)kv->sequences, (long long)heads);
    const int64_t need = hyena_attn_step_ws_bytes(kv->sequences, heads, kv->kv_heads, kv->head_dim);
    if (need > 0 && (!ws || ws_bytes < need))
        return hyena_fail(HYENA_EINVAL, "%s: workspace of %lld bytes, %lld needed", who, (long long)ws_bytes, (long long)need);
    a.q = (const char*)q->ptr;
    a.q_seq_stride = q->token_stride * 2;
    a.q_head_stride = q->head_stride * 2;
    a.lens = lens;
    a.out = (char*)out;
    a.scale = scale * 1.4426950408889634f;
    a.heads = (int32_t)heads;
    a.group = (int32_t)(heads / kv->kv_heads);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)(kv->sequences * heads));
#define AT_CASE(D, P)                                                                            \
    if (dtype == D && kv->dtype == P) hipLaunchKernelGGL((attn_step_kernel<D, P>), grid, dim3(256), 0, s, a);
    AT_CASE(HYENA_DTYPE_BF16, HYENA_DTYPE_BF16)
    AT_CASE(HYENA_DTYPE_F16, HYENA_DTYPE_F16)
    AT_CASE(HYENA_DTYPE_BF16, HYENA_DTYPE_F8E4M3)
    AT_CASE(HYENA_DTYPE_F16, HYENA_DTYPE_F8E4M3)
#undef AT_CASE
    return hyena_check_launch(who);
}
