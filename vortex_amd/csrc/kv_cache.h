// What the kernels of the paged key / value cache share: element types and the address of a position.
#pragma once
#include "common.h"

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;

template <int DT> struct KvElem;            // a stored or an activation element as float32, and back
template <> struct KvElem<HYENA_DTYPE_BF16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float get(raw r) { return bf_to_f(r); }
    static __device__ __forceinline__ raw put(float f) { return (raw)f_to_bf_bits(f); }
};
template <> struct KvElem<HYENA_DTYPE_F16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float get(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
    static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
};
template <> struct KvElem<HYENA_DTYPE_F8E4M3> {
    typedef uint8_t raw;
    static __device__ __forceinline__ float get(raw r) { return __builtin_amdgcn_cvt_f32_fp8((int)r, 0); }
    // round to nearest even; the instruction turns what lies beyond +-448 into NaN, so the value is clamped first
    // (NaN compares false both times and stays)
    static __device__ __forceinline__ raw put(float f) {
        f = f > 448.f ? 448.f : (f < -448.f ? -448.f : f);
        return (raw)(__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false) & 0xff);
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

static inline int64_t kv_elem_bytes(int dtype) { return dtype == HYENA_DTYPE_F8E4M3 ? 1 : 2; }

// Checks a cache description and fills its device copy; 0 or a HYENA_E* code.
int kv_pages_check(const hyena_kv_pages* kv, int dtype, KvPages* out, const char* who);
