// Attention of one new token per sequence over a paged key / value cache.
//
//   s_j = scale * <q, K_j>,  o = sum_j 2^(s_j - m) V_j / sum_j 2^(s_j - m)     (scale includes log2 e)
//
// Bound by the bytes of K and V: one multiply-add per stored element and query head.  Everything is laid out so that
// each wavefront streams pages through its registers without a barrier:
//   * S^T = K Q^T on v_mfma_f32_16x16x32: a lane holds 8 consecutive elements of ONE key (16 bytes as they lie in the
//     page), the columns are up to 16 query heads that share the key head;
//   * the result leaves key 4*(lane/16) + i of a 16-key piece in register i of lane `lane`, column lane % 16 -- which is
//     where the A operand of the next product wants the weights if its 32 keys are numbered (lane/16, piece, i).
//     So the weights never move between lanes;
//   * O = P V: a lane loads 8 consecutive elements of a value row for each of its 8 keys (full rows per 16 lanes) and
//     pairs the keys up with one v_perm per two elements.
// The weights go in as three 16-bit terms that hold all 24 bits of a float32 weight: the products are free beside the
// loads, and what is left between the output and the float32 formula is the order of the sums (with two terms, 16 bits in
// bf16, about one output in 2000 came out as a neighbour of the value it rounds to).
#include "kv_addr.h"
#include "kv_cache.h"

namespace {

constexpr int WAVES = 4;                    // wavefronts of a block (they share nothing)
constexpr int64_t STREAM_BYTES = 128 << 20; // reads beyond this are non-temporal, unless rows share pages

struct AttnArgs {
    KvPages kv;
    const char* q;
    int64_t q_seq_stride, q_head_stride;    // bytes
    const int32_t* lens;
    char* out;
    float* part_o;                          // [2 * wavefronts][heads of a tile][HDP]
    float* part_ml;                         // [2 * wavefronts][heads of a tile][2]
    int32_t* runs;                          // [sequences][key heads][query tiles][2]: first and last wavefront of a row
    float scale;                            // includes log2(e): the softmax works in powers of two
    int32_t heads, group, qtiles;           // query heads per key head, in tiles of 16
    int32_t waves;                          // of the even cut
};

// Weights are 2^(score - m + SHIFT), m a whole number that follows the scores up when one exceeds it by more than LAZY, so
// that changing m scales the sums without a rounding.  float16 terms end at 2^-24, 2^-35 of a weight at m.  There m
// follows the scores down as well, once all of a tile's lie more than LOW below it, so that a long row of small weights is
// not rounded away behind one large one: a tile's weights are kept to 2^-28 of its largest.  m stays within DEEP of the
// largest score, which keeps the sums below 2^100.
template <int DT> struct Mma;
template <> struct Mma<HYENA_DTYPE_BF16> {
    static constexpr float LAZY = 8.f, SHIFT = 0.f, LOW = 0.f, DEEP = 0.f;
    static __device__ __forceinline__ f32x4 dot(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf2(lo, hi); }
    // Weights x, y >= 0 as the exact sum of three terms, none of them 0 unless the weight is, so that a weight times an
    // infinite value stays infinite instead of adding 0 * inf.  A term is the largest bf16 number BELOW what is left (its
    // predecessor cut off), which leaves 1..2^16 and then 1..2^8 units of the weight's last place.
    static __device__ __forceinline__ uint32_t below(float x, float y) {
        return __builtin_amdgcn_perm(__builtin_elementwise_sub_sat(__float_as_uint(y), 1u),
                                     __builtin_elementwise_sub_sat(__float_as_uint(x), 1u), 0x07060302u);
    }
    static __device__ __forceinline__ void split(float x, float y, bool, uint32_t (&t)[3]) {
        t[0] = below(x, y);
        x -= bf_lo(t[0]), y -= bf_hi(t[0]);
        t[1] = below(x, y);
        t[2] = pack(x - bf_lo(t[1]), y - bf_hi(t[1]));
    }
    template <bool HI> static __device__ __forceinline__ uint32_t from_f8(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
    }
};
template <> struct Mma<HYENA_DTYPE_F16> {
    static constexpr float LAZY = 4.f, SHIFT = 11.f, LOW = 8.f, DEEP = 32.f;
    typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 h2;
    static __device__ __forceinline__ f32x4 dot(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const h2 h = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(uint32_t, h);
    }
    // Head, rest and rest of the rest, cut off and the last one rounded: all bits of a weight down to 2^-24.  Beside
    // infinite values (`inf`) the terms of a weight above 0 are 2^-24 at least: a weight times an infinite value stays
    // infinite instead of adding 0 * inf.
    typedef __attribute__((__vector_size__(4))) uint16_t u16x2;
    static __device__ __forceinline__ void split(float x, float y, bool inf, uint32_t (&t)[3]) {
        const u16x2 least = {(uint16_t)(x > 0.f), (uint16_t)(y > 0.f)};
        const auto a = __builtin_amdgcn_cvt_pkrtz(x, y);
        x -= (float)a[0], y -= (float)a[1];
        const auto b = __builtin_amdgcn_cvt_pkrtz(x, y);
        t[0] = __builtin_bit_cast(uint32_t, a), t[1] = __builtin_bit_cast(uint32_t, b);
        t[2] = pack(x - (float)b[0], y - (float)b[1]);
        if (inf)                                // of numbers >= 0 the larger one has the larger bits
            for (uint32_t& z : t) z = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, z), least));
    }
    template <bool HI> static __device__ __forceinline__ uint32_t from_f8(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
    }
};

__device__ __forceinline__ int lane_id() { return __lane_id(); }
__device__ __forceinline__ float max_over_keys(float x) {       // over the four lanes lane, lane ^ 16, ^ 32, ^ 48
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_keys(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Tiles of TK positions, in the order (sequence, key head, query tile, position); where a tile index falls.
struct Place {
    int64_t total;          // tiles of all sequences
    int64_t waves;          // wavefronts that get some of them, one tile at least
    int64_t first;          // tiles ahead of sequence b
    int32_t b, tiles;       // the sequence and its tiles per (key head, query tile)
};

__device__ __forceinline__ int32_t seq_len(const AttnArgs& a, int32_t b) {
    return (int32_t)min((int64_t)max(a.lens[b], 0), a.kv.reach);
}

__device__ __forceinline__ int64_t scan64(int64_t x, int lane) {            // inclusive, over the lanes
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(x, o);
        x += lane >= o ? up : 0;
    }
    return x;
}
__device__ __forceinline__ int64_t of_lane(int64_t x, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane), hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), lane);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Sums the tiles of all sequences, each lane those of consecutive ones, and finds the sequence that holds the first
// tile of wavefront w: its lane first, then among that lane's.
__device__ __forceinline__ Place find_place(const AttnArgs& a, int tk_shift, int32_t rows, int64_t w) {
    const int lane = lane_id();
    const int64_t B = a.kv.sequences, per = (B + 63) / 64;
    auto tiles = [&](int64_t b) { return b < B ? ((int64_t)seq_len(a, (int32_t)b) + (1 << tk_shift) - 1) >> tk_shift : 0; };
    Place p = {0, 0, 0, 0, 0};
    int64_t mine = 0;
    for (int64_t i = 0; i < per; ++i) mine += tiles(lane * per + i);
    const int64_t incl = scan64(mine, lane);
    p.total = of_lane(incl, 63) * rows;
    p.waves = min(p.total, (int64_t)a.waves);
    if (w >= p.waves) return p;
    const int64_t goal = kv_first_tile(w, p.total, p.waves);
    const int l = __builtin_ctzll(__ballot(incl * rows > goal));
    int64_t ahead = of_lane(incl, l) - of_lane(mine, l);                    // in tiles per (key head, query tile)
    if (per == 1) {
        p.b = l;
        p.tiles = (int32_t)of_lane(mine, l);
        p.first = ahead * rows;
        return p;
    }
    for (int64_t i = 0; i < per; i += 64) {
        const int64_t t = i + lane < per ? tiles(l * per + i + lane) : 0, sum = scan64(t, lane);
        const uint64_t hit = __ballot((ahead + sum) * rows > goal);
        if (hit) {
            const int k = __builtin_ctzll(hit);
            p.b = (int32_t)(l * per + i + k);
            p.tiles = (int32_t)of_lane(t, k);
            p.first = (ahead + of_lane(sum, k) - p.tiles) * rows;
            return p;
        }
        ahead += of_lane(sum, 63);
    }
    return p;
}

template <int DT, bool F8, int HDP, bool PAD>
struct Walk {
    typedef Mma<DT> M;
    static constexpr int NC = HDP / 32;                             // 32-element pieces of a row
    static constexpr int DL = HDP >= 128 ? 8 : HDP / 16;            // value elements of a lane, per block of 16 lanes
    static constexpr int VB = HDP > 128 ? HDP / 128 : 1;            // such blocks in a row
    static constexpr int NT = F8 ? (HDP >= 256 ? 1 : HDP == 128 ? 2 : 4) : (HDP >= 128 ? 1 : HDP == 64 ? 2 : 4);
    static constexpr int TK = 32 * NT, TK_SHIFT = NT == 1 ? 5 : NT == 2 ? 6 : 7;
    static constexpr bool K16 = F8 && !PAD && HDP >= 64;            // e4m3 keys in 16-byte pieces
    static constexpr int KW = F8 ? 2 : 4, VW = F8 ? (DL >= 4 ? DL / 4 : 1) : DL / 2;   // dwords of a key / value piece
    static constexpr int ES = F8 ? 1 : 2;
    // The products want consecutive lanes on different keys (and 8-bit values 8 bytes a lane): requests like that are
    // slow in the address unit (e4m3: 5.0 against 5.9 TB/s).  So rows are requested in 64 consecutive 16-byte pieces and
    // turned around in an LDS buffer of the wavefront, 16 rows at a time, two buffers in turn.  Piece x of row y lies at
    // x ^ row_swizzle(y), which spreads the reads over the banks.  (LDS operations of a wavefront stay in order.)
    static constexpr int RB = HDP * ES, CPR = RB / 16;              // bytes and 16-byte pieces of a row
    static constexpr bool TURN = !PAD && CPR >= 4, TURNV = TURN && F8;
    static constexpr int LDS_BYTES = TURN ? 2 * 16 * RB : 0;        // of a wavefront
    static __device__ __forceinline__ int row_swizzle(int row) { return (RB >= 256 ? row : row / (256 / RB)) & (CPR - 1) & 15; }

    // What a tile belongs to (wave-uniform).
    struct Tile {
        int32_t b, kh, qt, tile, n;         // sequence, key head, query tile, tile of the row, positions of the sequence
    };

    const AttnArgs& a;
    int lane, r, j;                         // lane, lane % 16, lane / 16
    Tile at;                                // the tile that is requested next, or was last
    int32_t ent_b, ent, ent0;               // 64 entries of the table row of sequence ent_b, one a lane, from entry ent0 on
    uint32_t koff[TURN ? CPR / 4 : 1], voff[TURNV ? CPR / 4 : 1];   // lane's bytes in a 16-key piece
    char* lds;                              // this wavefront's part of the LDS
    uint32_t kmask;                         // PAD: bit c: piece c of this lane is inside the row
    u32x4 q[NC], qn[NC];                    // query heads of the row at work, and of the one requested
    int32_t pg[2 * NT];                     // pages of the requested tile's 16-key pieces
    uint32_t kr[TURN ? 1 : NT][2][NC][KW], vr[NT][8][VB][VW];
    u32x4 kt[TURN ? 2 * NT : 1][TURN ? CPR / 4 : 1], vt[TURNV ? 2 * NT : 1][TURNV ? CPR / 4 : 1];
    f32x4 o[VB * DL];
    float m, mx, l;                         // the weights' reference, the largest score it has followed, their sum

    __device__ __forceinline__ Walk(const AttnArgs& args, char* buf) : a(args), lds(buf) {
        lane = lane_id();
        r = lane & 15;
        j = lane >> 4;
        ent_b = -1;
        const int hd = a.kv.head_dim;
        if constexpr (TURN) {
#pragma unroll
            for (int i = 0; i < CPR / 4; ++i) {
                const int row = (64 * i + lane) / CPR, x = 16 * (lane % CPR ^ row_swizzle(row));
                koff[i] = row * (uint32_t)a.kv.k.slot_stride + x;
                if constexpr (TURNV) voff[i] = row * (uint32_t)a.kv.v.slot_stride + x;
            }
        } else {
            koff[0] = r * (uint32_t)a.kv.k.slot_stride + (PAD ? 0 : 8 * ES * j);
        }
        const int vd = VB > 1 ? 8 * r : DL * r;
        if (!TURNV) voff[0] = 4 * j * (uint32_t)a.kv.v.slot_stride + (!PAD || vd < hd ? vd * ES : 0);
        kmask = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) kmask |= !PAD || key_dim(c) < hd ? 1u << c : 0;
    }
    // First element of the 8 that this lane holds of a key row in step c of the product.
    __device__ __forceinline__ int key_dim(int c) const { return K16 ? 64 * (c / 2) + 16 * j + 8 * (c % 2) : 32 * c + 8 * j; }

    __device__ __forceinline__ void load_q() {
        const int head = at.qt * 16 + r;
        const char* p = a.q + at.b * a.q_seq_stride + (int64_t)(at.kh * a.group + (head < a.group ? head : 0)) * a.q_head_stride;
#pragma unroll
        for (int c = 0; c < NC; ++c) qn[c] = *(const u32x4*)(p + (!PAD || kmask >> c & 1 ? 2 * key_dim(c) : 0));
    }
    __device__ __forceinline__ void start(int32_t qt) {             // of a row: its heads, nothing summed yet
        const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NC; ++c) q[c] = qt * 16 + r < a.group && (!PAD || kmask >> c & 1) ? qn[c] : zero;
        nothing();
    }
    __device__ __forceinline__ void nothing() {
#pragma unroll
        for (int i = 0; i < VB * DL; ++i) o[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        m = mx = -INFINITY;
        l = 0.f;
    }

    // Whether the m of some head has to move for a tile of which `top` is this lane's largest score; and moves it, for
    // all heads of the tile at once.
    __device__ __forceinline__ bool off(float top) const {
        bool move = __any(top > m + M::LAZY);
        if constexpr (M::LOW > 0) {
            uint64_t low = __ballot(top < m - M::LOW && m > mx - M::DEEP);      // in all four lanes of a head
            low &= low >> 32;
            move |= (low & low >> 16 & 0xffff) != 0;
        }
        return move;
    }
    __device__ __forceinline__ void follow(float top) {
        const float t = ceilf(max_over_keys(top));
        mx = fmaxf(mx, t);
        const float mn = M::LOW > 0 ? fmaxf(t, mx - M::DEEP) : mx;
        const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));      // a power of two, without a rounding
        m = mn;
        l *= f;
        const f32x4 g = {__shfl(f, 4 * j), __shfl(f, 4 * j + 1), __shfl(f, 4 * j + 2), __shfl(f, 4 * j + 3)};
#pragma unroll
        for (int i = 0; i < VB * DL; ++i) o[i] *= g;
    }

    // Whether a value of the tile may be infinite (float16; bf16 weights need no care, e4m3 has no infinities).
    __device__ __forceinline__ bool infinite() const {
        if constexpr (F8 || DT != HYENA_DTYPE_F16) return false;
        else {
            typename M::u16x2 top = {0, 0};
#pragma unroll
            for (int g = 0; g < NT; ++g)
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int b = 0; b < VB; ++b)
#pragma unroll
                        for (int w = 0; w < VW; ++w)
                            top = __builtin_elementwise_max(top, __builtin_bit_cast(typename M::u16x2, vr[g][i][b][w] & 0x7fff7fffu));
            return __any(top[0] >= 0x7c00 || top[1] >= 0x7c00);
        }
    }

    // Page of a 16-key piece (wave-uniform), or -1.
    __device__ __forceinline__ int32_t page_of(int32_t key0) {
        const int32_t e = key0 >> a.kv.page_shift;
        if (ent_b != at.b || (uint32_t)(e - ent0) >= 64u) {
            ent_b = at.b;
            ent0 = e;
            const int64_t i = (int64_t)e + lane, last = ((int64_t)at.n - 1) >> a.kv.page_shift;
            ent = i <= last ? a.kv.table[at.b * a.kv.table_stride + i] : -1;
            asm volatile("" : "+v"(ent));       // wait for it here: a wait at its use would hold up every tile
        }
        return kv_page_or_none(key0 < at.n ? __builtin_amdgcn_readlane(ent, e - ent0) : -1, a.kv.num_pages);
    }
    __device__ __forceinline__ void pages() {
#pragma unroll
        for (int s = 0; s < 2 * NT; ++s) pg[s] = page_of(at.tile * TK + 16 * s);
    }

    template <bool STREAM, class T> static __device__ __forceinline__ T fetch(const char* p) {
        if constexpr (STREAM) return __builtin_nontemporal_load((const T*)p);
        else return *(const T*)p;
    }
    template <bool STREAM, int W> static __device__ __forceinline__ void load(uint32_t (&to)[W], const char* p) {
        if constexpr (W == 4) {
            const u32x4 x = fetch<STREAM, u32x4>(p);
            to[0] = x[0], to[1] = x[1], to[2] = x[2], to[3] = x[3];
        } else if constexpr (W == 2) {
            const u32x2 x = fetch<STREAM, u32x2>(p);
            to[0] = x[0], to[1] = x[1];
        } else if constexpr (F8 && DL == 2) {
            to[0] = fetch<STREAM, uint16_t>(p);
        } else {
            to[0] = fetch<STREAM, uint32_t>(p);
        }
    }

    // A piece whose page is not there is read from page 0 and left out later.
    template <bool STREAM> __device__ __forceinline__ void load_keys() {
#pragma unroll
        for (int s = 0; s < 2 * NT; ++s) {
            const int32_t slot = (at.tile * TK + 16 * s) & ((1 << a.kv.page_shift) - 1);
            const char* base = a.kv.k.ptr + at.kh * a.kv.k.head_stride + (int64_t)max(pg[s], 0) * a.kv.k.page_stride + (int64_t)slot * a.kv.k.slot_stride;
            if constexpr (TURN) {
#pragma unroll
                for (int i = 0; i < CPR / 4; ++i) kt[s][i] = fetch<STREAM, u32x4>(base + koff[i]);
            } else {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint32_t d = PAD ? (kmask >> c & 1 ? (32 * c + 8 * j) * ES : 0) : 32 * c * ES;
                    load<STREAM, KW>(kr[s / 2][s % 2][c], base + (koff[0] + d));
                }
            }
        }
    }
    template <bool STREAM> __device__ __forceinline__ void load_values() {
#pragma unroll
        for (int s = 0; s < 2 * NT; ++s) {
            const int32_t slot = (at.tile * TK + 16 * s) & ((1 << a.kv.page_shift) - 1);
            const char* base = a.kv.v.ptr + at.kh * a.kv.v.head_stride + (int64_t)max(pg[s], 0) * a.kv.v.page_stride + (int64_t)slot * a.kv.v.slot_stride;
            if constexpr (TURNV) {
#pragma unroll
                for (int i = 0; i < CPR / 4; ++i) vt[s][i] = fetch<STREAM, u32x4>(base + voff[i]);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < VB; ++b) {
                    const uint32_t d = PAD && VB > 1 ? (8 * r + 128 * b < a.kv.head_dim ? 128 * b * ES : 0) : 128 * b * ES;
                    load<STREAM, VW>(vr[s / 2][4 * (s % 2) + i][b], base + (int64_t)i * a.kv.v.slot_stride + (voff[0] + d));
                }
        }
    }
    // 16 rows into the buffer of piece s.
    __device__ __forceinline__ void turn(int s, const u32x4 (&rows)[CPR / 4 ? CPR / 4 : 1]) {
#pragma unroll
        for (int i = 0; i < CPR / 4; ++i) *(u32x4*)(lds + s % 2 * 16 * RB + i * 1024 + lane * 16) = rows[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");     // no instruction; other lanes read this
    }
    // The values of a tile, 8 bytes a lane: elements 8 * (lane % 16) .. of rows 4 * (lane / 16) + 0..3 of every piece.
    __device__ __forceinline__ void turn_values() {
        if constexpr (TURNV) {
#pragma unroll
            for (int s = 0; s < 2 * NT; ++s) {
                turn(s, vt[s]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int b = 0; b < VB; ++b) {
                        const int row = 4 * j + i, byte = VB > 1 ? 8 * r + 128 * b : DL * r;
                        const char* p = lds + s % 2 * 16 * RB + row * RB + 16 * (byte / 16 ^ row_swizzle(row)) + byte % 16;
                        if constexpr (VW == 2) {
                            const u32x2 x = *(const u32x2*)p;
                            vr[s / 2][4 * (s % 2) + i][b][0] = x[0], vr[s / 2][4 * (s % 2) + i][b][1] = x[1];
                        } else {
                            vr[s / 2][4 * (s % 2) + i][b][0] = *(const uint32_t*)p;
                        }
                    }
            }
        }
    }
    // The 8 elements of step c of a lane's key in 16-key piece s.
    __device__ __forceinline__ u32x4 key_step(int s, int c) const {
        u32x4 x;
        uint32_t w[KW];
        if constexpr (TURN) {
            const u32x4 y = *(const u32x4*)(lds + s % 2 * 16 * RB + r * RB + 16 * ((4 * (K16 ? c / 2 : c) + j) ^ row_swizzle(r)));
#pragma unroll
            for (int i = 0; i < KW; ++i) w[i] = y[K16 ? 2 * (c % 2) + i : i];
        } else {
#pragma unroll
            for (int i = 0; i < KW; ++i) w[i] = kr[s / 2][s % 2][c][i];
        }
        if constexpr (F8) {
            x[0] = M::template from_f8<false>(w[0]), x[1] = M::template from_f8<true>(w[0]);
            x[2] = M::template from_f8<false>(w[1]), x[3] = M::template from_f8<true>(w[1]);
        } else {
            x[0] = w[0], x[1] = w[1], x[2] = w[2], x[3] = w[3];
        }
        if (PAD) {
            const u32x4 zero = {0, 0, 0, 0};
            x = kmask >> c & 1 ? x : zero;
        }
        return x;
    }

    // `count` tiles from `at` on.  next() moves `at` on by one tile and says whether that is a new row; done(tile, from)
    // is called after the last tile here of every row, of which the tiles from `from` on are in the sums.  The next
    // tile is requested while this one is worked on, over the end of a row as well.
    template <bool STREAM, class Next, class Done>
    __device__ __forceinline__ void run(int32_t count, Next next, Done done) {
        pages();
        load_q();
        load_keys<STREAM>();
        load_values<STREAM>();
        bool fresh = true;
        int32_t from = 0;
        float kscale = 0.f;
        while (true) {
            const Tile t = at;
            uint32_t ok = 0;                        // pieces of the tile whose page is there
#pragma unroll
            for (int s = 0; s < 2 * NT; ++s) ok |= pg[s] >= 0 ? 1u << s : 0;
            const bool full = ok == (1u << (2 * NT)) - 1 && (t.tile + 1) * TK <= t.n;
            if (fresh) {
                start(t.qt);
                from = t.tile;
                kscale = a.scale * (a.kv.k.scale ? a.kv.k.scale[t.kh] : 1.f);
            }
            f32x4 s[2 * NT];
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                s[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
                if constexpr (TURN) turn(i, kt[i]);
#pragma unroll
                for (int c = 0; c < NC; ++c) s[i] = M::dot(key_step(i, c), q[c], s[i]);
            }
            if (--count > 0) fresh = next();        // behind the last tile: that one again, unused
            pages();
            if (fresh) load_q();
            load_keys<STREAM>();
            turn_values();
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][e] *= kscale;
            if (!full) {
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool in = (ok >> i & 1) && t.tile * TK + 16 * i + 4 * j + e < t.n;
                        s[i][e] = in ? s[i][e] : -INFINITY;
#pragma unroll
                        for (int b = 0; b < VB; ++b)
#pragma unroll
                            for (int w = 0; w < VW; ++w) vr[i / 2][4 * (i % 2) + e][b][w] = in ? vr[i / 2][4 * (i % 2) + e][b][w] : 0;
                    }
            }
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][e]);
            if (off(top)) follow(top);
            const float base = m == -INFINITY ? 0.f : m - M::SHIFT;
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[i][e] = __builtin_amdgcn_exp2f(s[i][e] - base);
                    l += s[i][e];
                }
            const bool inf = infinite();
#pragma unroll
            for (int g = 0; g < NT; ++g) {
                u32x4 p[3];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t t[3];
                    M::split(s[2 * g + e / 2][2 * (e % 2)], s[2 * g + e / 2][2 * (e % 2) + 1], inf, t);
                    p[0][e] = t[0], p[1][e] = t[1], p[2][e] = t[2];
                }
#pragma unroll
                for (int b = 0; b < VB; ++b)
#pragma unroll
                    for (int i = 0; i < DL; ++i) {
                        u32x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (F8) {
                                const uint32_t w = __builtin_amdgcn_perm(vr[g][2 * e + 1][b][i / 4], vr[g][2 * e][b][i / 4],
                                                                         i % 4 < 2 ? 0x05010400u : 0x07030602u);
                                x[e] = i % 2 ? M::template from_f8<true>(w) : M::template from_f8<false>(w);
                            } else {
                                x[e] = __builtin_amdgcn_perm(vr[g][2 * e + 1][b][i / 2], vr[g][2 * e][b][i / 2],
                                                             i % 2 ? 0x07060302u : 0x05040100u);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < 3; ++t) o[b * DL + i] = M::dot(p[t], x, o[b * DL + i]);
                    }
            }
            load_values<STREAM>();
            if (count == 0 || fresh) done(t, from);
            if (count == 0) return;
        }
    }

    // The finished row: every head of the tile divided by its sum, rounded and stored.
    __device__ __forceinline__ void store(const Tile& t) {
        typedef KvElem<DT> E;
        const float sum = sum_over_keys(l), vs = a.kv.v.scale ? a.kv.v.scale[t.kh] : 1.f;
        const float inv = sum != 0.f ? vs / sum : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 4 * j + e;
            const float f = __shfl(inv, row);
            if (t.qt * 16 + row >= a.group) continue;
            char* y = a.out + ((int64_t)t.b * a.heads + t.kh * a.group + t.qt * 16 + row) * a.kv.head_dim * 2;
#pragma unroll
            for (int v = 0; v < VB; ++v) {
                const int d = VB > 1 ? 8 * r + 128 * v : DL * r;
                if (PAD && d >= a.kv.head_dim) continue;
                uint32_t w[DL / 2];
#pragma unroll
                for (int i = 0; i < DL / 2; ++i) w[i] = M::pack(o[v * DL + 2 * i][e] * f, o[v * DL + 2 * i + 1][e] * f);
                if constexpr (DL == 8) *(u32x4*)(y + 2 * d) = (u32x4){w[0], w[1], w[2], w[3]};
                else if constexpr (DL == 4) *(u32x2*)(y + 2 * d) = (u32x2){w[0], w[1]};
                else *(uint32_t*)(y + 2 * d) = w[0];
            }
        }
    }

    // A part of a row, for the join: unnormalised sums, maximum and sum of the weights.
    __device__ __forceinline__ void store_part(int64_t slot, int32_t qt) {
        const int rows = min(a.group, 16);
        const float sum = sum_over_keys(l);
        if (j == 0 && qt * 16 + r < a.group) {
            float* ml = a.part_ml + (slot * rows + r) * 2;
            ml[0] = m;
            ml[1] = sum;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 4 * j + e;
            if (qt * 16 + row >= a.group) continue;
            float* y = a.part_o + (slot * rows + row) * HDP;
#pragma unroll
            for (int v = 0; v < VB; ++v)
#pragma unroll
                for (int i = 0; i < DL; ++i) y[(VB > 1 ? 8 * r + 128 * v : DL * r) + i] = o[v * DL + i][e];
        }
    }
};

// The tiles of all (sequence, key head, query tile) rows in one line, cut into equal runs, one per wavefront: lengths are
// on the device, and this is even for any of them.  A row inside one run is finished here; the first and the last row
// of a run may be parts (slots 2w and 2w + 1), which attn_join_kernel adds up.
// Measured, both launches: one sequence of 131072 keys, 32 heads of 128, bf16: 328 us, 6.5 TB/s of reads (7.0 is what
// reads alone reach); 64 sequences of 0..4096 keys: 367 us, 6.4 TB/s; 32 of up to 32768, 8 key heads, e4m3: 190 us,
// 6.0 TB/s; one of 2000 keys (33 MB): 14.8 us, of which 8 are two launches without work.
template <int DT, bool F8, int HDP, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, HDP > 128 ? 1 : 2) attn_walk_kernel(AttnArgs a) {
    typedef Walk<DT, F8, HDP, PAD> W;
    // few tiles are spread over all blocks: the first wavefronts of all blocks come first
    const int64_t w = (int64_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * gridDim.x + blockIdx.x;
    const int32_t rows = a.kv.kv_heads * a.qtiles;
    const Place p = find_place(a, W::TK_SHIFT, rows, w);
    if (w >= p.waves) return;
    const int64_t t0 = kv_first_tile(w, p.total, p.waves), t1 = kv_first_tile(w + 1, p.total, p.waves);
    int32_t row = (int32_t)((t0 - p.first) / p.tiles), tiles = p.tiles;
    __shared__ __align__(16) char lds[W::LDS_BYTES ? WAVES * W::LDS_BYTES : 16];
    W walk(a, lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * W::LDS_BYTES);
    walk.at = {p.b, row / a.qtiles, row % a.qtiles, (int32_t)(t0 - p.first - (int64_t)row * tiles), seq_len(a, p.b)};
    int64_t line = t0 - walk.at.tile;               // of the first tile of the row in `walk.at`
    int64_t base = line;                            // the same, of the row at work
    auto next = [&]() {
        if (++walk.at.tile < tiles) return false;
        walk.at.tile = 0;
        line += tiles;
        if (++walk.at.qt == a.qtiles) {
            walk.at.qt = 0;
            if (++walk.at.kh == a.kv.kv_heads) {
                walk.at.kh = 0;
                do {                                // another sequence has tiles: the run does not end here
                    ++walk.at.b;
                    walk.at.n = seq_len(a, walk.at.b);
                    tiles = (int32_t)(((int64_t)walk.at.n + W::TK - 1) >> W::TK_SHIFT);
                } while (tiles == 0);
            }
        }
        return true;
    };
    auto done = [&](const typename W::Tile& t, int32_t from) {
        const int32_t all = (int32_t)(((int64_t)t.n + W::TK - 1) >> W::TK_SHIFT);
        if (from == 0 && t.tile == all - 1) walk.store(t);
        else walk.store_part(2 * w + (from == 0), t.qt);
        if (from == 0 && walk.lane == 0) {
            int32_t* run = a.runs + (((int64_t)t.b * a.kv.kv_heads + t.kh) * a.qtiles + t.qt) * 2;
            run[0] = (int32_t)w;
            run[1] = (int32_t)(t.tile == all - 1 ? w : kv_wave_of_tile(base + all - 1, p.total, p.waves));
        }
        base = line;
    };
    // Rows that must share pages, since they count more positions than there are, find each other's reads in the caches
    // (bf16, 32 heads of 128: 4 rows of the same 131072 keys 570 us against 794 with non-temporal loads, 16 of 8192 149 /
    // 191, 2 of 32768 99 / 110; 3 of 32768 264 / 241).  In 8 bits they do not need them (16 of 32768, 8 key heads: 147 / 140).
    const bool shared = !F8 && p.total / rows * W::TK - (int64_t)a.kv.sequences * (W::TK - 1) > (int64_t)a.kv.num_pages << a.kv.page_shift;
    if (!shared && p.total * W::TK * a.kv.head_dim * 2 * W::ES > STREAM_BYTES * a.qtiles) walk.template run<true>((int32_t)(t1 - t0), next, done);
    else walk.template run<false>((int32_t)(t1 - t0), next, done);
}

// Short rows: one block per row, its wavefronts take the tiles in turn and add up their parts in LDS.  One launch, bound
// by its chain of latencies (table, keys, values): 203 keys of 32 heads 6.4 us; 256 keys, in a recorded graph, 6.6 us
// where the even cut takes 9.1.
template <int HDP> constexpr int short_waves() { return HDP > 128 ? 4 : 8; }

template <int DT, bool F8, int HDP, bool PAD>
__global__ void __launch_bounds__(64 * short_waves<HDP>()) attn_short_kernel(AttnArgs a) {
    typedef Walk<DT, F8, HDP, PAD> W;
    constexpr int N = short_waves<HDP>(), BYTES = W::LDS_BYTES > 16 * HDP * 4 ? W::LDS_BYTES : 16 * HDP * 4;
    __shared__ __align__(16) char lds[N * BYTES];               // to turn rows around, then [wavefront][head][HDP] sums
    __shared__ float ms[N][16], ls[N][16];
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t qt = blockIdx.x % a.qtiles, kh = blockIdx.x / a.qtiles % a.kv.kv_heads, b = blockIdx.x / a.qtiles / a.kv.kv_heads;
    const int32_t n = seq_len(a, b), tiles = (int32_t)(((int64_t)n + W::TK - 1) >> W::TK_SHIFT), hd = a.kv.head_dim;
    W walk(a, lds + wv * BYTES);
    walk.at = {b, kh, qt, wv, n};
    if (wv < tiles) {
        auto next = [&]() { walk.at.tile += N; return false; };
        auto done = [](const typename W::Tile&, int32_t) {};
        walk.template run<false>((tiles - wv + N - 1) / N, next, done);
    } else {
        walk.nothing();
    }
    const float sum = sum_over_keys(walk.l);
    if (walk.j == 0) ms[wv][walk.r] = walk.m, ls[wv][walk.r] = sum;
    __syncthreads();
    const int rows = min(a.group - qt * 16, 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int row = 4 * walk.j + e;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < N; ++w) top = fmaxf(top, ms[w][row]);
        const float f = __builtin_amdgcn_exp2f(ms[wv][row] - (top == -INFINITY ? 0.f : top));
        if (row >= rows) continue;
        float* y = (float*)lds + (wv * 16 + row) * HDP;
#pragma unroll
        for (int v = 0; v < W::VB; ++v)
#pragma unroll
            for (int i = 0; i < W::DL; ++i) y[(W::VB > 1 ? 8 * walk.r + 128 * v : W::DL * walk.r) + i] = walk.o[v * W::DL + i][e] * f;
    }
    __syncthreads();
    const float vs = a.kv.v.scale ? a.kv.v.scale[kh] : 1.f;
    for (int x = tid; x < rows * HDP; x += 64 * N) {
        const int row = x / HDP, d = x % HDP;
        if (d >= hd) continue;
        float top = -INFINITY, s = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < N; ++w) top = fmaxf(top, ms[w][row]);
        top = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < N; ++w) {
            s += ls[w][row] * __builtin_amdgcn_exp2f(ms[w][row] - top);
            v += ((const float*)lds)[(w * 16 + row) * HDP + d];
        }
        typedef KvElem<DT> E;
        ((typename E::raw*)a.out)[((int64_t)b * a.heads + kh * a.group + qt * 16 + row) * hd + d] = E::put(s != 0.f ? v * (vs / s) : 0.f);
    }
}

// Rows that lie in several runs: the parts of one head weighted by 2^(m - max), every GROUPS-th added up by one group of
// lanes, then the groups'.  THREADS work on one head and request up to 32 (256 threads, heads of 128) of its parts at
// once.  Sequences without a position get zeros here.
template <int DT, int HDP, int THREADS>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
    constexpr int VL = HDP / 4, GROUPS = THREADS / VL, AHEAD = 4;   // lanes of a part, parts at a time, and in flight
    __shared__ __align__(16) float acc[256 / THREADS][GROUPS][HDP];
    __shared__ float tot[256 / THREADS][GROUPS], mx[256 / THREADS][GROUPS];
    const int sub = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, grp = tid / VL, d = tid % VL * 4;
    const int64_t item = (int64_t)blockIdx.x * (256 / THREADS) + sub;
    const bool there = item < (int64_t)a.kv.sequences * a.heads;
    const int32_t b = there ? (int32_t)(item / a.heads) : 0, head = there ? (int32_t)(item % a.heads) : 0;
    const int32_t kh = head / a.group, in = head % a.group, hd = a.kv.head_dim, gr = min(a.group, 16);
    typedef KvElem<DT> E;
    typename E::raw* y = (typename E::raw*)a.out + ((int64_t)b * a.heads + head) * hd;
    const int32_t* run = a.runs + (((int64_t)b * a.kv.kv_heads + kh) * a.qtiles + in / 16) * 2;
    const int32_t n = seq_len(a, b), w0 = run[0], w1 = run[1];
    if (there && n == 0)
        for (int i = tid; i < hd; i += THREADS) y[i] = 0;
    const bool join = there && n > 0 && w0 < w1;
    auto slot = [&](int32_t w) { return (int64_t)(2 * w + (w == w0)) * gr + in % 16; };
    float m = -INFINITY, sum = 0.f;                 // of this group's parts
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int32_t w = w0 + grp; join && w <= w1; w += GROUPS * AHEAD) {
        f32x4 v[AHEAD];
        float pm[AHEAD], ps[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int64_t s = slot(min(w + GROUPS * i, w1));
            v[i] = *(const f32x4*)(a.part_o + s * HDP + d);
            pm[i] = a.part_ml[s * 2], ps[i] = a.part_ml[s * 2 + 1];
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) top = w + GROUPS * i <= w1 ? fmaxf(top, pm[i]) : top;
        const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m - base);
        m = top;
        sum *= old;
        x *= old;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (w + GROUPS * i > w1) continue;
            const float f = __builtin_amdgcn_exp2f(pm[i] - base);
            sum += f * ps[i];
            x += v[i] * f;
        }
    }
    if (join) {
        *(f32x4*)&acc[sub][grp][d] = x;
        if (d == 0) tot[sub][grp] = sum, mx[sub][grp] = m;
    }
    __syncthreads();
    if (!join) return;
    float top = -INFINITY, s = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, mx[sub][g]);
    top = top == -INFINITY ? 0.f : top;
    float f[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        f[g] = __builtin_amdgcn_exp2f(mx[sub][g] - top);
        s += f[g] * tot[sub][g];
    }
    const float vs = a.kv.v.scale ? a.kv.v.scale[kh] : 1.f, inv = s != 0.f ? vs / s : 0.f;
    for (int i = tid; i < hd; i += THREADS) {
        float v = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) v += f[g] * acc[sub][g][i];
        y[i] = E::put(v * inv);
    }
}

int padded(int64_t hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

// Whether every row is short: what the table can name (lengths are on the device) keeps a block's wavefronts at a few
// tiles each, and the blocks are few enough to run at once or nearly.  Even cut against this form in us, calls in a recorded
// graph:                          heads of 128, bf16   64, bf16      64, float16   128, e4m3
//   32 rows of 128 KiB               9.1 /  6.6         9.6 /  7.5    9.8 /  7.7   10.1 /  7.8
//   32 rows of 512 KiB              11.8 / 11.3        13.0 / 14.5   12.8 / 14.7   13.6 / 16.9
//   32 rows of 1 MiB                14.0 / 16.6        14.9 / 22.6   14.8 / 23.3   15.9 / 27.5
//   128 rows of 512 KiB             19.5 / 14.4        19.2 / 16.0   19.5 / 16.5   20.0 / 18.4
//   512 rows of 32 KiB              12.5 / 10.6        12.6 / 10.7   12.8 / 11.1   13.2 / 12.1
//   512 rows of 512 KiB             50.9 / 49.8        49.1 / 53.1   48.8 / 53.8   50.8 / 52.3
//   1024 rows of 32 KiB             13.4 / 18.7        13.7 / 18.7   13.9 / 19.4   14.8 / 21.8
//   2048 rows of 32 KiB             18.1 / 32.3        18.9 / 33.7   19.5 / 34.8   20.4 / 40.1
// The border of 512 KiB is that of heads of 128 in bf16; the others lose up to 4 us at it with few rows or many.
bool short_rows(const hyena_kv_pages* kv, int64_t heads) {
    const int64_t ov = hyena_override(HYENA_OV_ATTN_SHORT);
    if (ov >= 0) return ov != 0;
    const int64_t rows = kv->sequences * kv->kv_heads * ((heads / kv->kv_heads + 15) / 16);
    const int64_t bytes = kv->table_width * kv->page_size * kv->head_dim * 2 * kv_elem_bytes(kv->dtype);   // of a row
    return bytes <= (512 << 10) && rows <= 512;
}

// Wavefronts of the even cut.  One per SIMD leaves fewer parts to join: 2000 keys of 32 heads in bf16 14.3 us against 16.3
// with two, 8000 keys 31.7 / 31.5, 32768 keys 87 / 92, 8 sequences of 2048 48 / 53, 16 of 4096 and 8191 with 4 key heads of
// 64 in float16 20.0 / 21.1 and 32.6 / 33.2, 32 of 4096 with 8 key heads in e4m3 54 / 59; equal on long rows (131072 keys
// 335 / 332).  With many rows each wavefront changes rows often, and a second one on the SIMD works meanwhile (2048 rows of
// up to 4096 keys: 385 us against 390 with one).
int64_t waves_for(const hyena_kv_pages* kv, int64_t heads) {
    const int64_t rows = kv->sequences * kv->kv_heads * ((heads / kv->kv_heads + 15) / 16);
    return kv->head_dim <= 128 && rows > 1024 ? 2048 : 1024;
}

template <int DT, bool F8, int HDP, bool PAD>
void launch(const AttnArgs& a, bool few, hipStream_t s) {
    if (few) {
        hipLaunchKernelGGL((attn_short_kernel<DT, F8, HDP, PAD>), dim3((unsigned)a.kv.sequences * a.kv.kv_heads * a.qtiles),
                           dim3(64 * short_waves<HDP>()), 0, s, a);
        return;
    }
    hipLaunchKernelGGL((attn_walk_kernel<DT, F8, HDP, PAD>), dim3(a.waves / WAVES), dim3(64 * WAVES), 0, s, a);
    // many heads have few parts each: one wavefront a head instead of a block (2048 sequences of 32
    // keys, 32 heads on 8: 123 us with the walk, 80 with a wavefront: 67 for the walk, 13 for the join)
    const int64_t heads = (int64_t)a.kv.sequences * a.heads;
    if (heads > 1024) hipLaunchKernelGGL((attn_join_kernel<DT, HDP, 64>), dim3((unsigned)((heads + 3) / 4)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_join_kernel<DT, HDP, 256>), dim3((unsigned)heads), dim3(256), 0, s, a);
}

template <int DT, bool F8>
void launch_dim(const AttnArgs& a, bool pad, bool few, hipStream_t s) {
    switch (padded(a.kv.head_dim)) {
        case 32: return pad ? launch<DT, F8, 32, true>(a, few, s) : launch<DT, F8, 32, false>(a, few, s);
        case 64: return pad ? launch<DT, F8, 64, true>(a, few, s) : launch<DT, F8, 64, false>(a, few, s);
        case 128: return pad ? launch<DT, F8, 128, true>(a, few, s) : launch<DT, F8, 128, false>(a, few, s);
        default: return pad ? launch<DT, F8, 256, true>(a, few, s) : launch<DT, F8, 256, false>(a, few, s);
    }
}

}  // namespace

extern "C" int64_t hyena_attn_step_ws_bytes(const hyena_kv_pages* kv, int64_t heads) {
    if (!kv || kv->sequences <= 0 || heads <= 0 || kv->kv_heads <= 0 || kv->head_dim <= 0 || kv->head_dim > 256 || heads % kv->kv_heads)
        return 0;
    if (short_rows(kv, heads)) return 0;
    const int64_t g = heads / kv->kv_heads, rows = g < 16 ? g : 16;
    return 2 * waves_for(kv, heads) * rows * (padded(kv->head_dim) + 2) * 4 +
           kv->sequences * kv->kv_heads * ((g + 15) / 16) * 8;
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
    if (((uintptr_t)out & 15)) return hyena_fail(HYENA_EALIGN, "%s: out must be 16-byte aligned", who);
    KvHeads qh;
    if ((rc = kv_heads_check(q, true, "q", kv->sequences, heads, &qh, who))) return rc;
    // a lane's place in a 16-key piece is a 32-bit offset
    if (a.kv.k.slot_stride < 0 || a.kv.v.slot_stride < 0 || a.kv.k.slot_stride > (1 << 27) || a.kv.v.slot_stride > (1 << 27))
        return hyena_fail(HYENA_ENOSUP, "%s: positions of a page that lie %lld bytes apart", who, (long long)a.kv.k.slot_stride);
    const int64_t need = hyena_attn_step_ws_bytes(kv, heads);
    const bool few = short_rows(kv, heads);
    // a block of up to 512 threads per (sequence, key head, query tile), or 64 threads per (sequence, head)
    if (kv->sequences * heads > KV_GRID_THREADS / (few ? 512 : 64) - 4)
        return hyena_fail(HYENA_EINVAL, "%s: %lld sequences of %lld heads are too many for one call", who,
                          (long long)kv->sequences, (long long)heads);
    if (!few && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
        return hyena_fail(HYENA_EINVAL, "%s: workspace of %lld bytes (16-byte aligned), %lld needed", who, (long long)ws_bytes,
                          (long long)need);
    a.q = qh.ptr;
    a.q_seq_stride = qh.token_stride;
    a.q_head_stride = qh.head_stride;
    a.lens = lens;
    a.out = (char*)out;
    a.scale = scale * 1.4426950408889634f;
    a.heads = (int32_t)heads;
    a.group = (int32_t)(heads / kv->kv_heads);
    a.qtiles = (a.group + 15) / 16;
    a.waves = (int32_t)waves_for(kv, heads);
    a.part_o = (float*)ws;
    a.part_ml = a.part_o + 2 * (int64_t)a.waves * (a.group < 16 ? a.group : 16) * padded(kv->head_dim);
    a.runs = (int32_t*)(a.part_ml + 4 * (int64_t)a.waves * (a.group < 16 ? a.group : 16));
    const bool f8 = kv->dtype == HYENA_DTYPE_F8E4M3;
    // the plain form loads 16 bytes of a row at a time and whole rows; other row lengths and, in 8 bits, strides that
    // are only 8-byte multiples take the form that loads 8 bytes and masks the pieces behind a row's end
    const bool pad = kv->head_dim != padded(kv->head_dim) ||
                     (f8 && ((kv->k.page_stride | kv->k.head_stride | kv->k.slot_stride | kv->v.page_stride | kv->v.head_stride |
                              kv->v.slot_stride) & 15));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == HYENA_DTYPE_BF16) f8 ? launch_dim<HYENA_DTYPE_BF16, true>(a, pad, few, s) : launch_dim<HYENA_DTYPE_BF16, false>(a, pad, few, s);
    else f8 ? launch_dim<HYENA_DTYPE_F16, true>(a, pad, few, s) : launch_dim<HYENA_DTYPE_F16, false>(a, pad, few, s);
    return hyena_check_launch(who);
}
