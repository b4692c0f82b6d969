// What the two kernels of attention over the paged int8 K/V cache share: the
// arguments, the cut of the work into equal ranges, the halves of an operand.
#pragma once

#include <math.h>

#include "kz_cache.cuh"

namespace kz {

constexpr int kKT = 128;                    // keys a tile
constexpr int kMinTiles = 4;                // tiles a CTA's range has at least
constexpr int kTreeWords = KZ_TREE_MAX_NODES / 32;

struct CacheAttArgs {
    CacheView c;
    SeqView s;
    const float* q;
    int64_t q_bs, q_rs;
    const int32_t* counts;
    const int32_t* parents;
    int64_t parents_bs;
    float* out;
    float* parts;          // two slots a CTA: sums [RT][D], maxima [RT], weights [RT]; NULL: every range is whole
    int batch, tokens, heads, group;
    float scale;
    int* status;
};

// ------------------------------------------------------------- the schedule

// A sequence's share of the work.
struct Seq {
    int len, count, tiles, row_tiles;
};
template <int RT>
__device__ __forceinline__ Seq sequence(const CacheAttArgs& a, int b) {
    Seq s;
    const int64_t most = (int64_t)a.s.cols * a.c.page;
    s.len = (int)min((int64_t)max(0, a.s.lengths[b]), most);
    s.count = a.counts ? max(0, min(a.counts[b], a.tokens)) : a.tokens;
    s.tiles = (int)(((int64_t)s.len + s.count + kKT - 1) / kKT);
    s.row_tiles = (int)(((int64_t)s.count * a.group + RT - 1) / RT);
    return s;
}
// (the host refuses calls of 2^31 units or more)
__device__ __forceinline__ int units_of(const CacheAttArgs& a, const Seq& s) {
    return s.row_tiles * a.c.heads * (a.parts ? s.tiles : 1);            // whole ranges: a unit is a row tile
}
__device__ __forceinline__ int units_a_cta(const CacheAttArgs& a, int total, int ctas) {
    return max((int)(((int64_t)total + ctas - 1) / ctas), a.parts ? kMinTiles : 1);
}

// Sum of a value over the 128 threads that share `sum` (named barrier 1).
__device__ __forceinline__ int sum_128(int v, int* sum) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = v;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    return sum[0] + sum[1] + sum[2] + sum[3];
}

// A part of one (sequence, head, row tile): key tiles [t0, t1).
struct Segment {
    int b, h, rt, t0, t1;
    int len, count;
    int first_token, last_token;   // of the row tile
    bool whole;                    // all of its tiles
};

// Walks the segments of units [at, end): b0, base: the sequence that holds `at` and its first unit.
template <int RT>
struct Walk {
    int at, end, base, b;
    Seq s;
    __device__ __forceinline__ bool next(const CacheAttArgs& a, Segment& g) {
        if (at >= end) return false;
        while (at >= base + units_of(a, s)) {
            if (b + 1 >= a.batch) return false;
            base += units_of(a, s);
            s = sequence<RT>(a, ++b);
        }
        const int off = at - base;
        const int per = a.parts ? s.tiles : 1;
        const int hr = off / per;
        g.b = b;
        g.h = hr / s.row_tiles;
        g.rt = hr % s.row_tiles;
        g.t0 = off % per;
        const int take = min(per - g.t0, end - at);
        g.whole = take == per;
        g.t1 = a.parts ? g.t0 + take : s.tiles;
        at += take;
        g.len = s.len;
        g.count = s.count;
        g.first_token = g.rt * RT / a.group;
        g.last_token = min(s.count - 1, (g.rt * RT + RT - 1) / a.group);
        g.t1 = min(g.t1, (g.len + g.last_token) / kKT + 1);   // later tiles: no row of this tile sees them
        return true;
    }
};

// ------------------------------------------------------- codes and halves

// Two of a word's four codes (offset by 128) as fp16: the byte in the mantissa
// of 1024, less 1152.
template <int SEL>
__device__ __forceinline__ uint32_t two_codes(uint32_t w) {
    const uint32_t m = __byte_perm(w, 0x64646464u, SEL);
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// x's 11 leading bits; the rest, x less them, is exact
__device__ __forceinline__ float leading(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFFE000u); }
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// exp2(m - top), 0 where m is -inf (no key yet)
__device__ __forceinline__ float shrink(float m, float top) { return m == -INFINITY ? 0.0f : exp2_approx(m - top); }
__device__ __forceinline__ float pow2_field(int field) { return __uint_as_float((uint32_t)field << 23); }

// A row's weights times vs go to the tensor cores as fp16 halves; their largest
// is brought to 2^kLift by measuring the softmax's exponent from the running
// maximum of s + log2(vs), not of s alone (the sum of the weights is measured
// from it too, so it cancels).  vs counts as within 2^-100 .. 2^100 here, which
// keeps the weights themselves within fp32.
constexpr float kLift = 14.0f;
__device__ __forceinline__ float log2_vs(float vs) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(vs));
    return r != r ? r : fminf(fmaxf(r, -100.0f), 100.0f);
}

// The kernel for many rows (kz_cache_attention_tc.cu): tiles of kTcRows rows,
// one CTA a SM.
constexpr int kTcRows = 128;
int launch_cache_attention_tc(const CacheAttArgs& a, int d, int grid, cudaStream_t s);

}  // namespace kz
