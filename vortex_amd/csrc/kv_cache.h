// What the kernels of the paged key / value cache share: element types and the address of a position.
#pragma once
#include "common.h"

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;

template <int DT> struct KvElem;            // a stored or an activation element as float32, and back
template <> struct KvElem<HYENA_DTYPE_BF16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ raw put(float f) { return (raw)f_to_bf_bits(f); }
    static __device__ __forceinline__ float lo(uint32_t w) { return bf_lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf_hi(w); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf2(lo, hi); }
};
template <> struct KvElem<HYENA_DTYPE_F16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float get(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
    static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
    static __device__ __forceinline__ float lo(uint32_t w) { return get((raw)w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return get((raw)(w >> 16)); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return put(lo) | (uint32_t)put(hi) << 16; }
};
template <> struct KvElem<HYENA_DTYPE_F8E4M3> {
    // round to nearest even; the instruction turns what lies beyond +-448 into NaN, so the value is clamped first
    // (NaN compares false both times and stays)
    static __device__ __forceinline__ float clamp(float f) { return f > 448.f ? 448.f : (f < -448.f ? -448.f : f); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {         // two values in the low 16 bits
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamp(a), clamp(b), 0, false) & 0xffffu;
    }
};

struct KvSide {
    char* ptr;
    int64_t page_stride, head_stride, slot_stride;      // bytes
    const float* scale;
};

struct KvPages {
    KvSide k, v;
    const int32_t* table;
    int64_t table_stride;
    int32_t num_pages, kv_heads, head_dim;
    int32_t page_shift, sequences;
    int64_t reach;                                      // positions a table row can name
};

struct KvHeads {
    char* ptr;
    int64_t token_stride, head_stride;                  // bytes
};

constexpr int64_t KV_GRID_THREADS = (1LL << 32) - 1;   // of a launch in one dimension

static inline int64_t kv_elem_bytes(int dtype) { return dtype == HYENA_DTYPE_F8E4M3 ? 1 : 2; }

// Checks a cache description and fills its device copy; 0 or a HYENA_E* code.
int kv_pages_check(const hyena_kv_pages* kv, int dtype, KvPages* out, const char* who);
int kv_heads_check(const hyena_heads* h, bool required, const char* name, int64_t tokens, int64_t heads, KvHeads* out,
                   const char* who);
