// Paged key / value cache: rotary positions with the append, and page copies.
#include <algorithm>

#include "kv_addr.h"
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
    if (kv->table_width > (1LL << 30) / kv->page_size)
        return hyena_fail(HYENA_ENOSUP, "%s: a table row of %lld pages names more than 2^30 positions", who, (long long)kv->table_width);
    const int64_t es = kv_elem_bytes(kv->dtype);
    const hyena_kv_side* in[2] = {&kv->k, &kv->v};
    KvSide* to[2] = {&out->k, &out->v};
    for (int i = 0; i < 2; ++i) {
        hyena_kv_side s = *in[i];
        if (kv->num_pages == 1) s.page_stride = 0;
        if (kv->kv_heads == 1) s.head_stride = 0;
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

int kv_heads_check(const hyena_heads* h, bool required, const char* name, int64_t tokens, int64_t heads, KvHeads* out,
                   const char* who) {
    *out = {nullptr, 0, 0};
    if (!h || !h->ptr) return required ? hyena_fail(HYENA_EINVAL, "%s: %s is required", who, name) : 0;
    const int64_t ts = tokens == 1 ? 0 : h->token_stride, hs = heads == 1 ? 0 : h->head_stride;
    if (((uintptr_t)h->ptr & 15) || ts % 8 || hs % 8)
        return hyena_fail(HYENA_EALIGN, "%s: %s must be 16-byte aligned with strides of a multiple of 8 elements", who, name);
    *out = {(char*)h->ptr, ts * 2, hs * 2};
    return 0;
}

namespace {

struct Role {                               // the rows of q, k or v in a block's work
    KvHeads src, dst;                       // dst.ptr NULL: no rows of activations are written
    uint32_t heads, magic;                  // magic = ceil(2^32 / heads): i / heads = (i * magic) >> 32 for i * heads < 2^32
};

struct AppendArgs {
    KvPages kv;
    Role role[3];                           // q, k, v
    const int32_t *pos, *seq;
    const double* turns;
    int64_t tokens;
    int32_t half, per_seq, zero_skipped;    // half = rotary_dim / 2
    int32_t block_tokens, block_rounds;     // what a block takes: tokens, and rounds over their heads
};

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_TOKENS = 16;           // of a block at most: 16 * 128 pairs fill the LDS tables
constexpr int BATCH = 4;                    // pieces a thread has in flight

// VEC elements of an activation row as float32, and back.
template <int DT, int VEC, bool STREAM> struct Piece {
    typedef KvElem<DT> E;
    static constexpr int W = VEC >= 2 ? VEC / 2 : 1;
    uint32_t w[W];
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (VEC == 8) {
            const u32x4 x = STREAM ? __builtin_nontemporal_load((const u32x4*)p) : *(const u32x4*)p;
            w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
        } else if constexpr (VEC == 2) w[0] = *(const uint32_t*)p;
        else w[0] = *(const uint16_t*)p;
    }
    __device__ __forceinline__ void get(float (&x)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = i % 2 ? E::hi(w[i / 2]) : E::lo(w[i / 2]);
    }
    static __device__ __forceinline__ void put(char* p, const float (&x)[VEC]) {
        uint32_t o[W];
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = E::pack(x[2 * i], x[(2 * i + 1) % VEC]);
        if constexpr (VEC == 8) {
            const u32x4 v = {o[0], o[1], o[2], o[3]};
            if constexpr (STREAM) __builtin_nontemporal_store(v, (u32x4*)p);
            else *(u32x4*)p = v;
        }
        else if constexpr (VEC == 2) *(uint32_t*)p = o[0];
        else *(uint16_t*)p = (uint16_t)o[0];
    }
    static __device__ __forceinline__ void put_f8(char* p, const float (&x)[VEC], float scale) {
        typedef KvElem<HYENA_DTYPE_F8E4M3> P;
        uint32_t o[W];
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = P::pack(x[2 * i] / scale, x[(2 * i + 1) % VEC] / scale);
        if constexpr (VEC == 8) {
            const u32x2 v = {o[0] | o[1] << 16, o[2] | o[3] << 16};
            if constexpr (STREAM) __builtin_nontemporal_store(v, (u32x2*)p);
            else *(u32x2*)p = v;
        }
        else if constexpr (VEC == 2) *(uint16_t*)p = (uint16_t)o[0];
        else *(uint8_t*)p = (uint8_t)o[0];
    }
};

// Bound by its bytes: every element is read once and written once.  A block takes a few tokens.  A row of a head is cut
// into pieces: VEC pairs (half layout: two pieces, i and i + half; interleaved: one piece of VEC/2 pairs), or VEC
// elements behind the rotary part; a thread always works on the same piece of a row, neighbouring threads on
// neighbouring pieces, then neighbouring heads, so a wavefront moves whole rows.  Rounds go over the (token, head) rows of
// q, then k, then v: what a round works on is uniform, which keeps its addresses in scalar registers.  The first BATCH
// rounds are requested before the block makes the cosines and sines of its tokens in LDS (one pair a thread: an angle
// in float64 costs as much as rotating a dozen heads).  The angle is rounded to float32 once it is reduced to half a turn:
// off by at most pi 2^-24, and the result by as much of the pair's length, where the last rounding takes 2^-8 (float16 2^-11).
// Measured: 8192 tokens, 32 heads of 128 with their keys and values, dense keys too, bf16: 80-85 us, 5.5-5.9 TB/s read and
// written; one token 4.5 us.
template <int DT, bool F8, int VEC, bool IL, bool STREAM>
__global__ void __launch_bounds__(APPEND_THREADS) rotary_append_kernel(AppendArgs a) {
    typedef Piece<DT, VEC, STREAM> X;
    __shared__ __align__(16) float cs[APPEND_TOKENS * 128], sn[APPEND_TOKENS * 128];
    __shared__ int64_t offs[2][APPEND_TOKENS];      // bytes of the token's slot in the pages of k and v, -1: not written
    __shared__ int32_t skip[APPEND_TOKENS];
    const int tid = threadIdx.x, half = a.half, hd = a.kv.head_dim;
    const int64_t t0 = (int64_t)blockIdx.x * a.block_tokens;
    const int nt = (int)min((int64_t)a.block_tokens, a.tokens - t0);
    if (!a.zero_skipped) {                          // a block of padding rows reads none of them
        bool any = false;
        for (int i = 0; i < nt; ++i) any |= a.pos[t0 + i] >= 0;
        if (!any) return;
    }
    const int np = IL ? 2 * half / VEC : half / VEC, per_head = np + (hd - 2 * half) / VEC;
    const int slots = APPEND_THREADS / per_head, u = tid % per_head, s0 = tid / per_head;
    const bool rot = u < np;
    const int i0 = (rot || IL) ? u * VEC : 2 * half + (u - np) * VEC;       // the piece, and with pairs apart its partner
    const int i1 = i0 + half;
    const int rq = (nt * (int)a.role[0].heads + slots - 1) / slots, rk = (nt * (int)a.role[1].heads + slots - 1) / slots;
    const int r0 = blockIdx.y * a.block_rounds, r1 = min(r0 + a.block_rounds, rq + 2 * rk);
    X x[BATCH], y[BATCH];
    int row[BATCH], tok[BATCH];
    auto request = [&](int first) {
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            const int w = first + n, r = w < rq ? 0 : (w < rq + rk ? 1 : 2);
            const Role& role = a.role[r];
            const uint32_t i = (uint32_t)(w - (r == 0 ? 0 : (r == 1 ? rq : rq + rk))) * slots + s0;
            tok[n] = role.magic ? __umulhi(i, role.magic) : i;
            row[n] = w < r1 && s0 < slots && tok[n] < nt ? (int)(i - tok[n] * role.heads) : -1;
            if (row[n] >= 0) {
                const char* p = role.src.ptr + t0 * role.src.token_stride + 2 * i0 +
                                (uint32_t)(tok[n] * (uint32_t)role.src.token_stride + row[n] * (uint32_t)role.src.head_stride);
                x[n].load(p);
                if (!IL && rot) y[n].load(p + 2 * half);
            }
        }
    };
    request(r0);
    for (int i = tid; i < nt * half; i += APPEND_THREADS) {
        const int64_t pos = a.pos[t0 + i / half];
        const double turn = (double)pos * a.turns[i % half];
        sincospif(2.f * (float)(turn - rint(turn)), &sn[i], &cs[i]);
    }
    if (tid < nt) {
        const int64_t t = t0 + tid, pos = a.pos[t], s = a.seq ? a.seq[t] : t / a.per_seq;
        int64_t page = -1;
        if (s >= 0 && s < a.kv.sequences)
            page = kv_page_of(a.kv.table + s * a.kv.table_stride, a.kv.reach, a.kv.page_shift, a.kv.num_pages, pos);
        const int64_t slot = pos & ((1LL << a.kv.page_shift) - 1);
        offs[0][tid] = page < 0 ? -1 : page * a.kv.k.page_stride + slot * a.kv.k.slot_stride;
        offs[1][tid] = page < 0 ? -1 : page * a.kv.v.page_stride + slot * a.kv.v.slot_stride;
        skip[tid] = pos < 0;
    }
    __syncthreads();
    for (int first = r0; first < r1; first += BATCH) {
        if (first > r0) request(first);
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            if (row[n] < 0) continue;
            const int w = first + n, r = w < rq ? 0 : (w < rq + rk ? 1 : 2);
            const Role& role = a.role[r];
            float f0[VEC], f1[VEC];
            x[n].get(f0);
            if (!IL && rot) y[n].get(f1);
            if (rot && r < 2) {
                const float *c = cs + tok[n] * half + (IL ? i0 / 2 : i0), *s = sn + tok[n] * half + (IL ? i0 / 2 : i0);
                constexpr int N = IL ? VEC / 2 : VEC;
                float cc[N], ss[N];
                if constexpr (N % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        const f32x4 cv = *(const f32x4*)(c + i), sv = *(const f32x4*)(s + i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) cc[i + e] = cv[e], ss[i + e] = sv[e];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) cc[i] = c[i], ss[i] = s[i];
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float& e0 = IL ? f0[2 * i] : f0[i];
                    float& e1 = IL ? f0[2 * i + 1] : f1[i];
                    const float p0 = e0, p1 = e1;
                    e0 = p0 * cc[i] - p1 * ss[i];
                    e1 = p0 * ss[i] + p1 * cc[i];
                }
            }
            if (r < 2 && role.dst.ptr && (!skip[tok[n]] || (r == 0 && a.zero_skipped))) {
                char* p = role.dst.ptr + t0 * role.dst.token_stride + 2 * i0 +
                          (uint32_t)(tok[n] * (uint32_t)role.dst.token_stride + row[n] * (uint32_t)role.dst.head_stride);
                if (skip[tok[n]]) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f0[i] = f1[i] = 0.f;
                }
                X::put(p, f0);
                if (!IL && rot) X::put(p + 2 * half, f1);
            }
            if (r == 0) continue;
            const int64_t off = offs[r - 1][tok[n]];
            if (off < 0) continue;
            const KvSide& side = r == 1 ? a.kv.k : a.kv.v;
            char* p = side.ptr + off + (int64_t)row[n] * side.head_stride;
            const float sc = side.scale ? side.scale[row[n]] : 1.f;
            if constexpr (F8) {
                X::put_f8(p + i0, f0, sc);
                if (!IL && rot) X::put_f8(p + i1, f1, sc);
            } else {
                if (side.scale) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f0[i] /= sc, f1[i] /= sc;
                }
                X::put(p + 2 * i0, f0);
                if (!IL && rot) X::put(p + 2 * i1, f1);
            }
        }
    }
}

// One block per (pair, piece of the page, pool), N 16-byte requests a thread, all before the first store.  Bound by its
// bytes; non-temporal accesses, since nothing here is read twice.  N = 1 streams fastest (200 pages of 128 KB in 16
// pools: 135 us, 6.2 TB/s read and written, against 154 with N = 4), N = 4 needs fewer blocks where little is copied (a
// fork of one such page into 7: 4.6 against 5.5 us).
template <int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const char* src_base, int64_t src_pool, int64_t src_page, int64_t src_pages,
                                                         char* dst_base, int64_t dst_pool, int64_t dst_page, int64_t dst_pages,
                                                         int64_t bytes, int32_t pieces, const int32_t* src, const int32_t* dst,
                                                         int wide) {
    constexpr int64_t PIECE = 4096 * N;
    const int32_t pair = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const int64_t s = src[pair], d = dst[pair];
    if (s < 0 || s >= src_pages || d < 0 || d >= dst_pages) return;
    const char* from = src_base + (int64_t)blockIdx.y * src_pool + s * src_page + piece * PIECE;
    char* to = dst_base + (int64_t)blockIdx.y * dst_pool + d * dst_page + piece * PIECE;
    const int64_t n = min(PIECE, bytes - piece * PIECE);
    const int tid = threadIdx.x;
    if (wide && n == PIECE) {
        u32x4 x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __builtin_nontemporal_load((const u32x4*)from + tid + 256 * i);
#pragma unroll
        for (int i = 0; i < N; ++i) __builtin_nontemporal_store(x[i], (u32x4*)to + tid + 256 * i);
        return;
    }
    const int64_t n16 = wide ? n / 16 : 0;
    for (int64_t i = tid; i < n16; i += 256) ((u32x4*)to)[i] = ((const u32x4*)from)[i];
    for (int64_t i = 16 * n16 + tid; i < n; i += 256) to[i] = from[i];
}

template <int DT, bool F8, int VEC, bool IL, bool STREAM>
int launch_append(AppendArgs& a, hipStream_t s, const char* who) {
    // A block's rounds: up to 2 * BATCH over as many tokens as leave the fewest threads of a round idle, if that makes
    // enough blocks for every compute unit to hold a few (1024); else fewer, down to one round of one token a block
    // (the angles of a token are then made in several blocks, which costs less than waiting for one).
    const int64_t H = a.role[0].heads, K = a.role[1].heads;
    const int per_head = (IL ? 2 * a.half / VEC : a.half / VEC) + (a.kv.head_dim - 2 * a.half) / VEC;
    const int64_t slots = APPEND_THREADS / per_head;
    auto rounds = [&](int64_t nt) { return (nt * H + slots - 1) / slots + 2 * ((nt * K + slots - 1) / slots); };
    int64_t bt = 1;
    for (int64_t n = 2; n <= APPEND_TOKENS && rounds(n) <= 2 * BATCH && (a.tokens + n - 1) / n >= 1024; ++n)
        if (rounds(n) * bt <= rounds(bt) * n) bt = n;
    int64_t per = rounds(bt);
    const int64_t blocks = (a.tokens + bt - 1) / bt;
    if (blocks > KV_GRID_THREADS / APPEND_THREADS)
        return hyena_fail(HYENA_EINVAL, "%s: %lld tokens are too many for one call", who, (long long)a.tokens);
    const int64_t split = std::min<int64_t>(per, std::max<int64_t>((per + 2 * BATCH - 1) / (2 * BATCH), 1024 / blocks));
    per = (per + split - 1) / split;
    a.block_tokens = (int32_t)bt;
    a.block_rounds = (int32_t)per;
    hipLaunchKernelGGL((rotary_append_kernel<DT, F8, VEC, IL, STREAM>), dim3((unsigned)blocks, (unsigned)((rounds(bt) + per - 1) / per)),
                       dim3(APPEND_THREADS), 0, s, a);
    return hyena_check_launch(who);
}

template <int DT, bool F8>
int launch_append_type(AppendArgs& a, bool il, hipStream_t s, const char* who) {
    // Pieces of 8 elements where the rotary part allows them, of 2 or 1 where it ends elsewhere.  Non-temporal accesses
    // where the rows of q and k, read and written, are more than half of the last-level cache (8192 tokens of 96 rows of 128: 96.6
    // against 86.7 us); below, the rows stay there for the attention that follows (460 K rows of 64: 15.7 against 17.1).
    const int half = a.half;
    const bool stream = a.tokens * (a.role[0].heads + a.role[1].heads) * a.kv.head_dim * 4 > (128 << 20);
    if (il) {
        if (half % 4 == 0) return stream ? launch_append<DT, F8, 8, true, true>(a, s, who) : launch_append<DT, F8, 8, true, false>(a, s, who);
        return launch_append<DT, F8, 2, true, false>(a, s, who);
    }
    if (half % 8 == 0) return stream ? launch_append<DT, F8, 8, false, true>(a, s, who) : launch_append<DT, F8, 8, false, false>(a, s, who);
    if (half % 2 == 0) return launch_append<DT, F8, 2, false, false>(a, s, who);
    return launch_append<DT, F8, 1, false, false>(a, s, who);
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
    if (tokens < 0 || tokens >= (1LL << 31) || heads <= 0)
        return hyena_fail(HYENA_EINVAL, "%s: bad sizes tokens=%lld heads=%lld", who, (long long)tokens, (long long)heads);
    if (heads > 32768 || kv->kv_heads > 32768) return hyena_fail(HYENA_ENOSUP, "%s: more than 32768 heads", who);
    if (tokens == 0) return 0;
    const hyena_heads* in[3] = {q, k, v};
    const hyena_heads* to[3] = {q_out, k_out, nullptr};
    const char *in_name[3] = {"q", "k", "v"}, *to_name[3] = {"q_out", "k_out", ""};
    for (int i = 0; i < 3; ++i) {
        Role& r = a.role[i];
        const int64_t n = i == 0 ? heads : kv->kv_heads;
        if ((rc = kv_heads_check(in[i], true, in_name[i], tokens, n, &r.src, who)) ||
            (rc = kv_heads_check(to[i], i == 0, to_name[i], tokens, n, &r.dst, who)))
            return rc;
        for (const KvHeads* h : {&r.src, &r.dst})       // rows of a block's tokens are addressed with 32 bits
            if (h->token_stride < 0 || h->head_stride < 0 || APPEND_TOKENS * h->token_stride + n * h->head_stride >= (1LL << 32))
                return hyena_fail(HYENA_ENOSUP, "%s: rows of %s that lie %lld bytes apart", who, in_name[i],
                                  (long long)h->token_stride);
        if (r.dst.ptr && ((tokens > 1 && r.dst.token_stride == 0) || (n > 1 && r.dst.head_stride == 0)))
            return hyena_fail(HYENA_EINVAL, "%s: rows of %s share their memory", who, to_name[i]);
        r.heads = (uint32_t)n;
        r.magic = n == 1 ? 0 : (uint32_t)(((1ULL << 32) + n - 1) / n);
    }
    for (const hyena_kv_side* side : {&kv->k, &kv->v})
        if ((kv->num_pages > 1 && side->page_stride == 0) || (kv->kv_heads > 1 && side->head_stride == 0) || side->slot_stride == 0)
            return hyena_fail(HYENA_EINVAL, "%s: positions of the pages share their memory", who);
    if (!pos || (rotary_dim > 0 && !turns)) return hyena_fail(HYENA_EINVAL, "%s: pos and turns are required", who);
    if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > kv->head_dim)
        return hyena_fail(HYENA_EINVAL, "%s: rotary_dim %lld is not an even number up to head_dim %lld", who,
                          (long long)rotary_dim, (long long)kv->head_dim);
    if (!seq && (kv->sequences == 0 || tokens % kv->sequences))
        return hyena_fail(HYENA_EINVAL, "%s: without seq, tokens (%lld) must be a multiple of the sequences (%lld)", who,
                          (long long)tokens, (long long)kv->sequences);
    a.pos = pos;
    a.seq = seq;
    a.turns = turns;
    a.half = (int32_t)(rotary_dim / 2);
    a.per_seq = seq ? 1 : (int32_t)(tokens / kv->sequences);
    a.zero_skipped = zero_skipped != 0;
    a.tokens = tokens;
    hipStream_t s = (hipStream_t)stream;
    const bool f8 = kv->dtype == HYENA_DTYPE_F8E4M3, il = interleaved != 0;
    if (dtype == HYENA_DTYPE_BF16)
        return f8 ? launch_append_type<HYENA_DTYPE_BF16, true>(a, il, s, who) : launch_append_type<HYENA_DTYPE_BF16, false>(a, il, s, who);
    return f8 ? launch_append_type<HYENA_DTYPE_F16, true>(a, il, s, who) : launch_append_type<HYENA_DTYPE_F16, false>(a, il, s, who);
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
    if ((pools > 1 && dst_pools->pool_stride == 0) || (dst_pools->pages > 1 && dst_pools->page_stride == 0))
        return hyena_fail(HYENA_EINVAL, "%s: destination pages share their memory", who);
    const int64_t at = (int64_t)((uintptr_t)src_pools->base | (uintptr_t)dst_pools->base) |
                       (pools > 1 ? src_pools->pool_stride | dst_pools->pool_stride : 0) | src_pools->page_stride | dst_pools->page_stride;
    const int wide = (at & 15) == 0;
    const bool much = copies * pools > (64 << 20) / page_bytes;
    const int64_t piece = much ? 4096 : 16384, pieces = (page_bytes + piece - 1) / piece;
    constexpr int64_t MOST = KV_GRID_THREADS / 256;     // blocks of a launch; more pairs take several
    if (copies * pieces >= (1LL << 31) || pieces > MOST)
        return hyena_fail(HYENA_EINVAL, "%s: %lld copies of %lld bytes are too many for one call", who, (long long)copies,
                          (long long)page_bytes);
    for (int64_t done = 0; done < copies;) {
        const int64_t n = std::min(copies - done, MOST / pieces);
        hipLaunchKernelGGL(much ? copy_pages_kernel<1> : copy_pages_kernel<4>, dim3((unsigned)(n * pieces), (unsigned)pools),
                           dim3(256), 0, (hipStream_t)stream, (const char*)src_pools->base, src_pools->pool_stride,
                           src_pools->page_stride, src_pools->pages, (char*)dst_pools->base, dst_pools->pool_stride,
                           dst_pools->page_stride, dst_pools->pages, page_bytes, (int32_t)pieces, src + done, dst + done, wide);
        if (const int rc = hyena_check_launch(who)) return rc;
        done += n;
    }
    return 0;
}
