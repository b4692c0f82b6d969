// What the two kernels of attention over the paged int8 K/V cache share: the
// arguments, the cut of the work into equal ranges, the halves of an operand.
#pragma once

#include <math.h>

#include "kz_cache.cuh"

namespace kz {

constexpr int kKT = 128;                    // keys a tile
constexpr int kTcRows = 128;                // rows a tile of the kernel for many rows has
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
    float* parts;          // two slots a CTA: sums [RT][D], maxima [RT], weights (kSumUnit times) [RT]; NULL: no range ends inside a row tile
    int batch, tokens, heads, group;
    int ctas;              // the launch's
    FastDiv by_ctas;
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
// A call's work, summed over sequences (the host refuses calls of 2^31 units or
// more): its row tiles (of every head), their tiles of keys, and the most that a row tile has.
struct Work {
    int row_tiles, units, tiles;
    __device__ __forceinline__ void add(const CacheAttArgs& a, const Seq& s) {
        row_tiles += s.row_tiles * a.c.heads;
        units += s.row_tiles * a.c.heads * s.tiles;
        if (s.row_tiles) tiles = max(tiles, s.tiles);
    }
    __device__ __forceinline__ void add(const Work& o) {
        row_tiles += o.row_tiles;
        units += o.units;
        tiles = max(tiles, o.tiles);
    }
    __device__ __forceinline__ void add_warp() {
        row_tiles = __reduce_add_sync(0xffffffffu, row_tiles);
        units = __reduce_add_sync(0xffffffffu, units);
        tiles = __reduce_max_sync(0xffffffffu, tiles);
    }
};
// The units of each CTA, all having as many.
__device__ __forceinline__ int a_cta(const CacheAttArgs& a, int units) { return units > 0 ? div_by(units - 1, a.by_ctas) + 1 : 0; }

// Whether each CTA takes whole row tiles (a unit of work is then a row tile, not
// a tile of keys): where the most tiles that one would do that way are not more
// than in equal ranges, whose CTAs begin and end inside row tiles and leave parts
// to be joined, at the time of about three tiles.
// Measured whole / in ranges, up to 500, 700, 1000 and 2000 keys in 8 key heads
// of 128: single tokens of one sequence 10.0 / 9.0, 11.8 / 8.9, 14.2 / 8.6 and
// 21.5 / 9.7 us; of 8, 12.4 / 10.9, 14.6 / 10.4, 17.8 / 12.9 us; of 32, 12.9 /
// 16.2, -, 19.1 / 22.7, 31.0 / 31.3 us; of 64 (700) 27.2 / 30.4 us; chunks of 20
// tokens (80 rows) of one sequence 22.3 / 16.6, 24.1 / 16.6, 28.5 / 17.0 us, of
// 8 22.7 / 24.5, -, 28.9 / 26.4, of 16 24.2 / 33, -, 31 / 39, 47.7 / 50.2 us.
// Heads of 64 and 32 (1, 8 and 32 sequences of up to 700, 1500 and 4000 keys, 4 key
// heads; 1, 4, 7 and 64 rows): what it chooses is the better, or within 12% of it
// (32 of 700, one row, 64 wide 10.6 / 11.2, 32 wide 9.6 / 10.6), but for 64 rows over
// 32 of 1500: 31.6 / 36.5 and 28.7 / 31.1, where it takes ranges.
__device__ __forceinline__ bool whole_ranges(const CacheAttArgs& a, const Work& w) {
    return !a.parts || (int64_t)a_cta(a, w.row_tiles) * w.tiles <= (int64_t)a_cta(a, w.units) + 3;
}
__device__ __forceinline__ int units_of(const CacheAttArgs& a, const Seq& s, bool whole) {
    return s.row_tiles * a.c.heads * (whole ? 1 : s.tiles);
}

// A CTA's units [at, end), and the sequence that holds the first of them with that one's first unit.
struct Range {
    int at, end, b, base;
    bool whole;
};
struct RangeShared {
    Work warp[4];
    Work part[128];
    Range range;
};
// By 128 threads (named barrier 1); the result is in s.range for whoever syncs with them afterwards.
template <int RT>
__device__ __forceinline__ void find_range(const CacheAttArgs& a, RangeShared& s) {
    const int tid = threadIdx.x, each = (a.batch + 127) / 128;
    Work w{0, 0, 0};
    for (int b = tid * each; b < min(a.batch, (tid + 1) * each); ++b) {
        w.add(a, sequence<RT>(a, b));
        if (blockIdx.x == 0 && a.s.lengths[b] < 0) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
    }
    s.part[tid] = w;
    w.add_warp();
    if ((tid & 31) == 0) s.warp[tid >> 5] = w;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (tid != 0) return;
    w = s.warp[0];
    for (int i = 1; i < 4; ++i) w.add(s.warp[i]);
    Range r;
    r.whole = whole_ranges(a, w);
    const int total = r.whole ? w.row_tiles : w.units, per = a_cta(a, total);
    r.at = (int)min((int64_t)total, (int64_t)per * blockIdx.x);
    r.end = (int)min((int64_t)total, (int64_t)r.at + per);
    r.b = r.base = 0;
    if (r.at < r.end) {
        int i = 0;
        for (; i < 127; ++i) {
            const int n = r.whole ? s.part[i].row_tiles : s.part[i].units;
            if (r.at < r.base + n) break;
            r.base += n;
        }
        for (r.b = i * each; r.b < a.batch - 1; ++r.b) {
            const int n = units_of(a, sequence<RT>(a, r.b), r.whole);
            if (r.at < r.base + n) break;
            r.base += n;
        }
    }
    s.range = r;
}

// A part of one (sequence, head, row tile): key tiles [t0, t1).
struct Segment {
    int b, h, rt, t0, t1;
    int len, count;
    int first_token, last_token;   // of the row tile
    bool whole;                    // all of its tiles
};

// Walks the segments of a CTA's range.
template <int RT>
struct Walk {
    int at, end, b, base;
    bool whole;
    Seq s;
    __device__ __forceinline__ Walk(const CacheAttArgs& a, const Range& r)
        : at(r.at), end(r.end), b(r.b), base(r.base), whole(r.whole) {
        if (at < end) s = sequence<RT>(a, b);
    }
    __device__ __forceinline__ bool next(const CacheAttArgs& a, Segment& g) {
        if (at >= end) return false;
        while (at >= base + units_of(a, s, whole)) {
            if (b + 1 >= a.batch) return false;
            base += units_of(a, s, whole);
            s = sequence<RT>(a, ++b);
        }
        const int off = at - base;
        const int per = whole ? 1 : s.tiles;
        const int hr = off / per;
        g.b = b;
        g.h = hr / s.row_tiles;
        g.rt = hr % s.row_tiles;
        g.t0 = off % per;
        const int take = min(per - g.t0, end - at);
        g.whole = take == per;
        g.t1 = whole ? s.tiles : g.t0 + take;
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
// keeps a weight within 2^114; their sum is kept in units of 2^20 (an exact
// factor, taken by the multiply-add that adds a weight up), so that 2^31 of them
// stay below 2^126.
constexpr float kLift = 14.0f;
constexpr float kSumUnit = 9.5367431640625e-7f;         // 2^-20
// o over the weights' sum, `inverse` that of the sum as it is kept: in this
// order neither factor leaves fp32 at either end of vs
__device__ __forceinline__ float over_sum(float o, float inverse) { return (o * kSumUnit) * inverse; }
__device__ __forceinline__ float log2_vs(float vs) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(vs));
    return r != r ? r : fminf(fmaxf(r, -100.0f), 100.0f);
}

// The kernel for many rows (kz_cache_attention_tc.cu): one CTA a SM.
int launch_cache_attention_tc(const CacheAttArgs& a, int d, cudaStream_t s);

}  // namespace kz
