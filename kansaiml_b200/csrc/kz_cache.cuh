// The paged int8 K/V cache as the kernels see it (kz_cache.cu, kz_cache_attention.cu).
#pragma once

#include "kz_common.cuh"

namespace kz {

// Pools of pages: codes [pages][heads][page][d], scale [pages][heads][page]; index 0 is K, 1 is V.
struct CacheView {
    int8_t* codes[2];
    float* scale[2];
    int pages, heads, page, shift;   // page == 1 << shift
};

// A call's sequences: page numbers [batch, cols] and tokens already in the cache [batch].
struct SeqView {
    const int32_t* table;
    const int32_t* lengths;
    int cols;
};

// x / d for 0 <= x < 2^31 by one multiply-high.
struct FastDiv {
    uint32_t d, m, l;
};
inline FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while ((1ull << f.l) < d) ++f.l;
    f.m = (uint32_t)(((1ull << 32) * ((1ull << f.l) - d)) / d + 1);
    return f;
}
__device__ __forceinline__ uint32_t div_by(uint32_t x, const FastDiv& f) { return (__umulhi(f.m, x) + x) >> f.l; }

// Host checks; each returns KZ_OK or records why not (`who`: the entry point).
int cache_view(const kz_cache* c, const char* who, CacheView* v);
int seq_view(const int32_t* table, int64_t cols, const int32_t* lengths, int64_t batch, const char* who, SeqView* v);

// The page that holds position pos of sequence b, or -1 where the table has
// none: before 0, past the table, or a page number that is not in the pool.
__device__ __forceinline__ int page_of(const CacheView& c, const SeqView& s, int64_t b, int64_t pos) {
    const int64_t i = pos >> c.shift;
    if (pos < 0 || i >= s.cols) return -1;
    const int page = __ldg(s.table + b * s.cols + i);
    return (unsigned)page < (unsigned)c.pages ? page : -1;
}

}  // namespace kz
