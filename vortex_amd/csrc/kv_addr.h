// Where a position of a sequence lives in a paged cache.  Plain C++ as well as device code.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define KV_FN static __host__ __device__ __forceinline__
#else
#define KV_FN static inline
#endif

// A page id as the table holds it: itself where it names one of num_pages pages, -1 everywhere else.
KV_FN int32_t kv_page_or_none(int32_t id, int32_t num_pages) {
    return (uint32_t)id < (uint32_t)num_pages ? id : -1;
}

// The page of position pos in a table row that reaches `reach` positions; -1 where there is none.
KV_FN int32_t kv_page_of(const int32_t* row, int64_t reach, int page_shift, int32_t num_pages, int64_t pos) {
    if (pos < 0 || pos >= reach) return -1;
    return kv_page_or_none(row[pos >> page_shift], num_pages);
}

// Work of W <= T wavefronts over T tiles (one at least for each): wavefront w takes tiles [kv_first_tile(w), kv_first_tile(w + 1)).
KV_FN int64_t kv_first_tile(int64_t w, int64_t T, int64_t W) { return w * T / W; }
// The wavefront that takes tile t < T (the inverse of the line above).
KV_FN int64_t kv_wave_of_tile(int64_t t, int64_t T, int64_t W) { return ((t + 1) * W - 1) / T; }
