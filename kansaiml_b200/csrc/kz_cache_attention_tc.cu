// Attention over the paged int8 K/V cache for many rows (chunks of a prompt,
// trees over grouped heads): the same arithmetic as kz_cache_attention.cu --
// codes exact in fp16, q and the weights as two fp16 halves, a fresh sum per
// tile of keys -- on the tcgen05 tensor cores.
//
// A CTA works on 128 rows (of one key head) and walks tiles of 128 keys:
//   S[128 rows, 128 keys] = Qhi K^T + Qlo K^T     Q in tensor memory, K in shared memory
//   O[128 rows, d]        = Phi V + Plo V         P in tensor memory (over S), V in shared memory
// with K and V converted from codes to fp16 as they arrive, in one layout (rows
// of 64 values, 128-byte swizzle) that is K-major for the first product and
// N-major for the second.  Warps 0-7: softmax, two threads a row (64 keys of
// each tile, and half of the row's sums in registers, to which each tile's O is
// added); 8-11 convert the next tiles; 12 issues the MMAs, 13 loads the pages
// (bulk copies), 14 and 15 zero the padding's rows.  The MMAs of tile t + 1's
// scores run while tile t's softmax does.
//
// Measured, join included: 2 chunks of 500 tokens over 8192 keys, 16 heads over 4
// key heads of 128: 152 us = 910 TFLOP/s over both halves, 0.55 of the tensor
// cores' measured rate (heads of 64: 130 us, of 32: 111); trees of 24 tokens (96
// rows) over 8 contexts of 2500 to 5000, 8 key heads of 128: 51 us, of which the 13
// tiles a CTA are 27, the start and the changes of row tile about 14, the rest the
// join and the tail.  What bounds the tiles is the softmax's chain: one takes
// about 3900 cycles, of which the MMAs are 2050 and the exponentials 1024; with
// neither MMAs nor conversions four fifths of the time remain.  A row a thread
// with the two warpgroups on alternate tiles took 207 us instead of 157 (S is read
// twice from tensor memory, at 128 bytes a cycle), joining O between the weights'
// steps 165 (spills), sums in the converters' warps 192, O kept in tensor memory
// over 2 or 4 tiles with a CTA-wide vote on rescaling 169 to 172; four threads a
// row 159 instead of 151 (at d = 64 the same).
//
// Tensor memory (512 columns): Q halves 0..d-1, S / P of even tiles 128..255,
// of odd tiles 256..383, O 384..383+d.  One CTA a SM.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kz_cache_attention.cuh"

namespace kz {
namespace {

constexpr int kTcThreads = 512;
constexpr int kSoftmax = 256;             // threads of the softmax: two a row
constexpr uint32_t kTmS = 128, kTmO = 384;

template <int D>
struct Tc {
    static constexpr int SUB = D <= 64 ? 1 : 2;            // sub-tiles of 64 values
    static constexpr int TILE = SUB * kKT * 128;           // bytes of a K or V tile in fp16
    static constexpr int CODES = kKT * D;                  // and in codes
    static constexpr int SMEM = 4 * TILE + 4 * CODES + 4 * 5 * kKT * 4 + 1024;
};

// fp16 x fp16 -> fp32, M x N; bit 16: B is N-major
constexpr uint32_t idesc_f16(uint32_t m, uint32_t n, bool b_n_major) {
    return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// D[tmem] (+)= A[tmem] x B[smem]
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(idesc), "r"(add)
        : "memory");
}
// Rows of 128 bytes (64 values), 128-byte swizzle, read N-major: 64 values of N
// a row, 8 rows of K 1024 bytes apart (stride), the next 64 of N at `next`
// bytes (leading).
__device__ __forceinline__ uint64_t smem_desc_n_sw128(uint32_t addr, uint32_t next) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(next >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Pairs of fp32 values: one instruction for two, each rounded on its own.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t bits_pair(uint32_t a, uint32_t b) {
    return pair(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// The registers of a warpgroup: each of the four starts with what the launch
// gives it, the two of the softmax take from the others'.
constexpr int kRegsLaunch = 65536 / kTcThreads, kRegsSoftmax = 192, kRegsConvert = 72, kRegsIssue = 56;
static_assert(2 * kRegsSoftmax + kRegsConvert + kRegsIssue <= 4 * kRegsLaunch, "an increase would wait for ever");
template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// 16 codes as 16 fp16 values (two 16-byte words)
__device__ __forceinline__ void codes_to_fp16(uint4 w, uint4& lo, uint4& hi) {
    w.x ^= 0x80808080u;
    w.y ^= 0x80808080u;
    w.z ^= 0x80808080u;
    w.w ^= 0x80808080u;
    lo = make_uint4(two_codes<0x4140>(w.x), two_codes<0x4342>(w.x), two_codes<0x4140>(w.y), two_codes<0x4342>(w.y));
    hi = make_uint4(two_codes<0x4140>(w.z), two_codes<0x4342>(w.z), two_codes<0x4140>(w.w), two_codes<0x4342>(w.w));
}

// A tile of codes [128 keys][D] to fp16 sub-tiles [128 keys][64], 128-byte
// swizzle, by 128 threads: a key a thread, 16 codes at a time.  Turn s takes
// the 16 codes c = c0 ^ s, with c0 from the key so that in every turn eight
// neighbouring lanes read eight bank groups and write eight (D = 64: c0 =
// 0, 2, 3, 1 of key / 2; both c0 and c0 ^ key / 2 run through all four).
// Everything about a place is linear under exclusive or, the turns' part a
// constant.
template <int D>
__device__ __forceinline__ void convert_tile(const uint8_t* codes, uint8_t* tile, int key) {
    constexpr int CH = D / 16, N = CH < 4 ? CH : 4;      // every load of a batch before its stores
    const int c0 = D == 128 ? key & 7 : D == 64 ? (0x1320 >> (2 * (key & 6))) & 3 : (key >> 2) & 1;
    const uint8_t* from = codes + key * D;
    uint8_t* to = tile + key * 128;
    const uint32_t from0 = c0 * 16, to0 = (uint32_t)(c0 >> 2) * (kKT * 128) + ((2 * (c0 & 3)) ^ (key & 7)) * 16;
#pragma unroll
    for (int s0 = 0; s0 < CH; s0 += N) {
        uint4 w[N];
#pragma unroll
        for (int n = 0; n < N; ++n) w[n] = *reinterpret_cast<const uint4*>(from + (from0 ^ ((s0 + n) * 16)));
#pragma unroll
        for (int n = 0; n < N; ++n) {
            constexpr int T = kKT * 128;
            const uint32_t at = to0 ^ (((s0 + n) >> 2) * T + 32 * ((s0 + n) & 3));
            uint4 lo, hi;
            codes_to_fp16(w[n], lo, hi);
            *reinterpret_cast<uint4*>(to + at) = lo;
            *reinterpret_cast<uint4*>(to + (at ^ 16)) = hi;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1) cache_attention_tc_kernel(const CacheAttArgs a) {
    using T = Tc<D>;
    extern __shared__ uint8_t ca_smem[];
    uint8_t* k_tiles = ca_smem + (-smem_u32(ca_smem) & 1023u);       // an offset, so that accesses stay shared-memory ones
    uint8_t* v_tiles = k_tiles + 2 * T::TILE;
    uint8_t* codes = v_tiles + 2 * T::TILE;                          // [2][K, V][CODES]
    float* scales = reinterpret_cast<float*>(codes + 4 * T::CODES);  // [4][ks, vs][128] as loaded
    float* factors = scales + 8 * kKT;                               // [4][ks, vs, log2 vs][128]
    __shared__ __align__(8) uint64_t s_code_full[2], s_code_empty[2], s_k_full[2], s_k_empty[2], s_v_full[2], s_v_empty[2],
        s_s_full[2], s_p_full[2], s_q_full, s_o_full, s_o_empty;
    __shared__ uint32_t s_tmem, s_bad[4];
    __shared__ float s_top[2][2][kTcRows], s_l[2][kTcRows];      // exchanged between a row's two threads
    __shared__ uint32_t s_sees[kTcRows][kTreeWords];
    __shared__ int32_t s_parent[KZ_TREE_MAX_NODES];
    __shared__ RangeShared s_range;
    __shared__ int s_abort;

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // uniform: so are the roles' branches
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_code_full[i]), 1);
            mbar_init(smem_u32(&s_code_empty[i]), 4);
            mbar_init(smem_u32(&s_k_full[i]), 4);
            mbar_init(smem_u32(&s_k_empty[i]), 1);
            mbar_init(smem_u32(&s_v_full[i]), 4);
            mbar_init(smem_u32(&s_v_empty[i]), 1);
            mbar_init(smem_u32(&s_s_full[i]), 1);
            mbar_init(smem_u32(&s_p_full[i]), 8);
        }
        mbar_init(smem_u32(&s_q_full), 8);
        mbar_init(smem_u32(&s_o_full), 1);
        mbar_init(smem_u32(&s_o_empty), 8);
        s_abort = 0;
        fence_mbarrier_init();
    }
    if (warp == 12) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    griddep_wait();

    if (warp < 4) find_range<kTcRows>(a, s_range);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_launch_dependents();           // not before this CTA has its tensor memory: a dependent may take some
    constexpr uint32_t tmem = 0;           // where all 512 columns begin
    Walk<kTcRows> walk(a, s_range.range);
    Segment g;
    // bounded as mbar_wait is, with fewer registers
    auto wait = [&](uint64_t& bar, int phase, int sleep = 0) {
        const uint32_t at = smem_u32(&bar);
        uint32_t began = 0;
        for (uint32_t n = 0; !mbar_try_wait(at, phase & 1);) {
            if (sleep) __nanosleep(sleep);
            if ((++n & 63u) == 0) {
                if (*reinterpret_cast<volatile int*>(&s_abort)) break;
                const uint32_t now = (uint32_t)(globaltimer_ns() >> 20);      // about a millisecond
                if (began == 0) began = now | 1u;
                if (now - began > 1024u && now > began) {
                    record_status(a.status, KZ_ERR_DEVICE_TIMEOUT);
                    s_abort = 1;
                    break;
                }
            }
        }
    };
    auto arrive = [&](uint64_t& bar) {     // once a warp
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar));
    };

    if (warp >= 12) registers_down<kRegsIssue>();
    if (warp == 13) {
        // ---- the loader: a lane a page of the tile
        const int pages = kKT >> a.c.shift;
        int it = 0;
        while (walk.next(a, g)) {
            const int held = g.len + g.count;
            auto page_id = [&](int t) {
                const int64_t pos = (int64_t)t * kKT + ((int64_t)lane << a.c.shift);
                return lane < pages && t < g.t1 && pos < held ? page_of(a.c, a.s, g.b, pos) : -2;   // -2: none needed
            };
            int id = page_id(g.t0);
            for (int t = g.t0; t < g.t1; ++t, ++it) {
                const int next = page_id(t + 1);
                wait(s_code_empty[it & 1], (it >> 1) + 1, 100);
                const uint32_t there = __ballot_sync(0xffffffffu, id >= 0), bad = __ballot_sync(0xffffffffu, id == -1);
                const uint32_t full = smem_u32(&s_code_full[it & 1]);
                if (lane == 0) {
                    s_bad[it & 3] = bad;
                    if (bad) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
                    mbar_arrive_expect_tx(full, __popc(there) * a.c.page * (2 * D + 8));
                }
                __syncwarp();
                if (id >= 0) {
                    const int64_t row = ((int64_t)id * a.c.heads + g.h) << a.c.shift;
                    const int k0 = lane << a.c.shift;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        bulk_load(smem_u32(codes + (2 * (it & 1) + kv) * T::CODES + k0 * D), a.c.codes[kv] + row * D,
                                  a.c.page * D, full);
                        bulk_load(smem_u32(scales + (2 * (it & 3) + kv) * kKT + k0), a.c.scale[kv] + row, a.c.page * 4, full);
                    }
                }
                id = next;
            }
        }
    } else if (warp == 12) {
        // ---- the MMAs: tile t's scores, then tile t - 1's output.  The whole
        // warp walks, one elected lane issues (elect.sync tells the compiler that
        // it is one: an MMA issued under a lane test measured 215 cycles, not 64)
        constexpr uint32_t id_s = idesc_f16(128, kKT, false), id_o = idesc_f16(128, D, true);
        int it = 0, segment = 0, pending = -1;
        auto output = [&](int t) {
            wait(s_p_full[t & 1], t >> 1);
            wait(s_v_full[t & 1], t >> 1);
            if (t > 0) wait(s_o_empty, t - 1);
            tc_fence_after();
            // uniform, so that the descriptors are made in uniform registers
            const uint32_t odd = __shfl_sync(0xffffffffu, t & 1, 0);
            const uint32_t v = smem_u32(v_tiles) + odd * T::TILE, p = tmem + kTmS + odd * 128;
            if (elect_one()) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < kKT / 16; ++i)
                        tc_mma_f16_ts(tmem + kTmO, p + (i >> 1) * 32 + (1 - half) * 16 + (i & 1) * 8, smem_desc_n_sw128(v + i * 2048, kKT * 128), id_o,
                                      half | i);
                tc_commit(smem_u32(&s_o_full));
                tc_commit(smem_u32(s_v_empty) + 8 * odd);
            }
            __syncwarp();
        };
        bool more = true;
        int t = 0;
        g.t0 = g.t1 = 0;
        while (more || pending >= 0) {
            // the next tile, if there is one; where the rows change, q comes after the last tile's
            // softmax, so its output goes first
            bool first = t >= g.t1;
            while (more && t >= g.t1) {
                more = walk.next(a, g);
                t = g.t0;
            }
            first = first || !more;
#pragma unroll 1
            for (int step = 0; step < 3; ++step) {
                if (step == (first ? 0 : 2) && pending >= 0) {
                    output(pending);
                    if (first) wait(s_o_full, pending);
                    if (!more) {                         // every commit has arrived before this CTA can end
                        wait(s_k_empty[pending & 1], pending >> 1);
                        wait(s_v_empty[pending & 1], pending >> 1);
                    }
                    pending = -1;
                }
                if (step != 1 || !more) continue;
                if (first)
                    wait(s_q_full, segment++);
                else if (it >= 2)
                    wait(s_o_full, it - 2);              // P(it - 2), in S's place, is used
                wait(s_k_full[it & 1], it >> 1);
                tc_fence_after();
                const uint32_t odd = __shfl_sync(0xffffffffu, it & 1, 0);
                const uint32_t k = smem_u32(k_tiles) + odd * T::TILE;
                if (elect_one()) {
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
                            tc_mma_f16_ts(tmem + kTmS + odd * 128, tmem + (1 - half) * (D / 2) + i * 8,
                                          smem_desc_k_sw128(k + (i >> 2) * (kKT * 128) + (i & 3) * 32), id_s, half | i);
                    tc_commit(smem_u32(s_s_full) + 8 * odd);
                    tc_commit(smem_u32(s_k_empty) + 8 * odd);
                }
                __syncwarp();
            }
            if (more) {
                pending = it++;
                ++t;
            }
        }
    } else if (warp < 8) {
        // ---- softmax: threads r and r + 128 have row r of the tile, each 64 of its
        // keys and half of its sums
        registers_up<kRegsSoftmax>();
        const int row = tid & 127, half = tid >> 7;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        // the row's two threads are in warps w and w + 4: they exchange by a barrier of those two
        auto meet_pair = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory"); };
        auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmax) : "memory"); };
        int it = 0;
        bool first_segment = true;
        while (walk.next(a, g)) {
            const int R = g.rt * kTcRows + row;
            const bool is_row = R < g.count * a.group;
            const int token = R / a.group;
            float unit = 0.0f;                     // a score in S is this much of a power of 2
            if (g.t0 < g.t1) {
                // q times scale log2(e), its largest value brought into [2^13, 2^14), as two halves
                const float* src = a.q + g.b * a.q_bs + (int64_t)token * a.q_rs +
                                   ((int64_t)g.h * a.group + R % a.group) * D + half * (D / 2);
                float4 x[D / 8];
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    x[i] = is_row ? *reinterpret_cast<const float4*>(src + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (a.parents)
                    for (int j = tid; j <= g.last_token; j += kSoftmax) s_parent[j] = a.parents[g.b * a.parents_bs + j];
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
                s_l[half][row] = top;
                meet();
                top = fmaxf(top, s_l[half ^ 1][row]);
                const float f = a.scale * 1.4426950408889634f;
                const int ex = min(max((int)(__float_as_uint(fabsf(top * f)) >> 23), 30), 254);
                const float up = f * pow2_field(267 - ex);
                unit = pow2_field(ex - 13);
                // 16 values a step: 8 columns of each half
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 v = x[4 * c + i / 2];
                        const float u = (i & 1 ? v.z : v.x) * up, w = (i & 1 ? v.w : v.y) * up;
                        hi[i] = half2_bits(leading(u), leading(w));
                        lo[i] = half2_bits(u - leading(u), w - leading(w));
                    }
                    tmem_st_32x32b_x8(tmem + lanes + half * (D / 4) + 8 * c, hi);
                    tmem_st_32x32b_x8(tmem + lanes + D / 2 + half * (D / 4) + 8 * c, lo);
                }
                tc_wait_st();
                tc_fence_before();
                arrive(s_q_full);
                if (a.parents) {
                    if (tid <= g.last_token - g.first_token) {
#pragma unroll
                        for (int w = 0; w < kTreeWords; ++w) s_sees[tid][w] = 0;
                        for (int n = g.first_token + tid; n >= 0;) {
                            s_sees[tid][n >> 5] |= 1u << (n & 31);
                            const int parent = s_parent[n];
                            n = parent < n ? parent : -1;
                        }
                    }
                    meet();
                }
            }
            const uint64_t unit2 = pair(unit, unit);
            float m = -INFINITY, l = 0.0f, corr = 0.0f, corr_next = 0.0f;
            float o[D / 2];
#pragma unroll
            for (int i = 0; i < D / 2; ++i) o[i] = 0.0f;
            // a tile's output joins the row's sums, `corr` the softmax's rescaling since the tile before
            auto join = [&] {
#pragma unroll
                for (int c = 0; c < D / 32; c += 2) {
                    uint32_t r[2][16];
                    tmem_ld_32x32b_x16(tmem + lanes + kTmO + half * (D / 2) + 16 * c, r[0]);
                    if (c + 1 < D / 32) tmem_ld_32x32b_x16(tmem + lanes + kTmO + half * (D / 2) + 16 * c + 16, r[1]);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (16 * c + i < D / 2) o[16 * c + i] = fmaf(o[16 * c + i], corr, __uint_as_float(r[i >> 4][i & 15]));
                }
            };
            // a warp none of whose rows are rows keeps the others' pace and computes nothing
            const bool idle = g.rt * kTcRows + (warp & 3) * 32 >= g.count * a.group;
            // (one turn more than tiles: the last joins the last tile's output)
#pragma unroll 1
            for (int t = g.t0; t < g.t1 || t > g.t0; ++t, ++it) {
                if (t == g.t1 || idle) {
                    if (t < g.t1) {
                        wait(s_s_full[it & 1], it >> 1);
                        arrive(s_p_full[it & 1]);
                    }
                } else {
                    const ulonglong2* ks = reinterpret_cast<const ulonglong2*>(factors + 3 * (it & 3) * kKT + 64 * half);
                    const ulonglong2 *vs = ks + kKT / 4, *lv = vs + kKT / 4;     // pairs of fp32 values
                    const uint32_t s_at = tmem + lanes + kTmS + (it & 1) * 128 + 64 * half;
                    wait(s_s_full[it & 1], it >> 1);
                    tc_fence_after();
                    const uint32_t bad = s_bad[it & 3];
                    // whether a row of the tile does not see one of the keys
                    const bool masked = t * kKT + kKT > g.len + (a.parents ? 0 : g.first_token + 1) || bad;
                    // the keys of chunk c (32 keys) that this row sees, a bit each
                    auto seen = [&](int c) {
                        const int first = t * kKT + 32 * c - g.len;      // the chunk's place among the new tokens
                        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
                        if (!is_row) return 0u;
                        uint32_t s;
                        if (a.parents) {
                            const uint32_t* mine = s_sees[token - g.first_token];
                            s = below(-first);
                            if (first > -32 && first < 0) s |= mine[0] << -first;
                            if (first >= 0 && first < KZ_TREE_MAX_NODES) {
                                const int i = first >> 5;
                                s = mine[i] >> (first & 31);
                                if ((first & 31) && i + 1 < kTreeWords) s |= mine[i + 1] << (32 - (first & 31));
                            }
                        } else {
                            s = below(token + 1 - first);
                        }
                        for (uint32_t left = bad; left; left &= left - 1) {
                            const int p0 = ((__ffs(left) - 1) << a.c.shift) - 32 * c;   // a missing page's keys
                            s &= ~(below(p0 + a.c.page) & ~below(p0));
                        }
                        return s;
                    };
                    uint64_t z[32];                      // s * ks
                    {
                        uint32_t r[2][32];
                        tmem_ld_32x32b_x32(s_at, r[0]);
                        tmem_ld_32x32b_x32(s_at + 32, r[1]);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const ulonglong2 f = ks[j];
                            const int c = j >> 3, i = (4 * j) & 31;
                            z[2 * j] = mul2(bits_pair(r[c][i], r[c][i + 1]), f.x);
                            z[2 * j + 1] = mul2(bits_pair(r[c][i + 2], r[c][i + 3]), f.y);
                        }
                    }
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t sees = seen(2 * half + c);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                float x0, x1;
                                unpair(z[16 * c + j], x0, x1);
                                if (!((sees >> (2 * j)) & 1u)) x0 = -INFINITY;
                                if (!((sees >> (2 * j + 1)) & 1u)) x1 = -INFINITY;
                                z[16 * c + j] = pair(x0, x1);
                            }
                        }
                    }
                    float top[4] = {m, m, m, m};         // the largest of s + log2 vs
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const ulonglong2 e = lv[j];
                        float x[4];
                        unpair(fma2(z[2 * j], unit2, e.x), x[0], x[1]);
                        unpair(fma2(z[2 * j + 1], unit2, e.y), x[2], x[3]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], x[k]);
                    }
                    float m_new = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    s_top[it & 1][half][row] = m_new;
                    meet_pair();
                    m_new = fmaxf(m_new, s_top[it & 1][half ^ 1][row]);
                    const float ref = m_new == -INFINITY ? 0.0f : kLift - m_new;
                    const uint64_t ref2 = pair(ref, ref);
                    uint64_t sum[2] = {0, 0};
                    // the weights, and their halves times vs over each 32 keys' own columns of S (16 of
                    // leading halves, 16 of the rest)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float p0, p1;
                            unpair(fma2(z[8 * c + j], unit2, ref2), p0, p1);
                            const uint64_t p = pair(exp2_approx(p0), exp2_approx(p1));
                            const ulonglong2 f = vs[4 * c + (j >> 1)];
                            sum[j & 1] = add2(sum[j & 1], p);
                            const uint64_t w = mul2(p, j & 1 ? f.y : f.x);
                            unpair(w, p0, p1);
                            const float h0 = leading(p0), h1 = leading(p1);
                            float l0, l1;
                            unpair(sub2(w, pair(h0, h1)), l0, l1);
                            hi[j] = half2_bits(h0, h1);
                            lo[j] = half2_bits(l0, l1);
                        }
                        tmem_st_32x32b_x8(s_at + 32 * (c >> 1) + 8 * (c & 1), hi);
                        tmem_st_32x32b_x8(s_at + 32 * (c >> 1) + 16 + 8 * (c & 1), lo);
                    }
                    const float corr_new = shrink(m, m_new);
                    m = m_new;
                    float s0, s1;
                    unpair(add2(sum[0], sum[1]), s0, s1);
                    l = fmaf(l, corr_new, (s0 + s1) * kSumUnit);
                    tc_wait_st();
                    tc_fence_before();
                    arrive(s_p_full[it & 1]);
                    corr_next = corr_new;
                }
                if (t > g.t0) {
                    wait(s_o_full, it - 1);
                    tc_fence_after();
                    if (!idle) join();
                    tc_fence_before();
                    arrive(s_o_empty);
                }
                corr = corr_next;
                if (t == g.t1) break;
            }
            s_l[half][row] = l;
            meet();
            l += s_l[half ^ 1][row];
            // o over the sum by one factor, which stays a normal number up to a sum of 2^100; past that
            // (V scales near 2^-100) its 2^-20 is taken afterwards, from what was stored.  A second factor
            // on o itself, though after the loop, made the loop 7 us of 151 slower (attend_chunk).
            const bool far = g.whole && l > 1.2676506e30f;
            const float f = !g.whole ? 1.0f : l == 0.0f ? 0.0f : (far ? 1.0f : kSumUnit) / l;
            float* slot = g.whole ? nullptr
                                  : a.parts + (2 * (int64_t)blockIdx.x + (first_segment ? 0 : 1)) * (kTcRows * (D + 2));
            first_segment = false;
            if (is_row) {
                float* dst = half * (D / 2) +
                             (g.whole ? a.out + (((int64_t)g.b * a.tokens + token) * a.heads + g.h * a.group + R % a.group) * D
                                      : slot + row * D);
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<float4*>(dst + 4 * i) =
                        make_float4(o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f, o[4 * i + 3] * f);
                if (far)
#pragma unroll 1
                    for (int i = 0; i < D / 2; ++i) dst[i] *= kSumUnit;
            }
            if (!g.whole && half == 0) {
                slot[kTcRows * D + row] = m;
                slot[kTcRows * D + kTcRows + row] = l;
            }
            meet();                                // the exchanged values and the tree's rows are free again
        }
    } else if (warp < 12) {
        // ---- codes to fp16, and the keys' factors
        registers_down<kRegsConvert>();
        const int t128 = tid - kSoftmax;
        int it = 0;
        while (walk.next(a, g)) {
            for (int t = g.t0; t < g.t1; ++t, ++it) {
                wait(s_code_full[it & 1], it >> 1);
                const float* raw = scales + 2 * (it & 3) * kKT;
                float* made = factors + 3 * (it & 3) * kKT;
                const bool out = t * kKT + t128 > g.len + g.last_token || ((s_bad[it & 3] >> (t128 >> a.c.shift)) & 1u);
                // a vs that is not finite reaches whoever sees the key through its score
                const float vs = out ? 0.0f : raw[kKT + t128];
                const bool fine = fabsf(vs) < INFINITY;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    wait(kv ? s_v_empty[it & 1] : s_k_empty[it & 1], (it >> 1) + 1);
                    if (kv == 0) {
                        made[t128] = fine ? raw[t128] : __uint_as_float(0x7FC00000u);
                        made[kKT + t128] = fine ? vs : 0.0f;
                        made[2 * kKT + t128] = log2_vs(fine ? vs : 0.0f);
                    }
                    convert_tile<D>(codes + (2 * (it & 1) + kv) * T::CODES, (kv ? v_tiles : k_tiles) + (it & 1) * T::TILE, t128);
                    fence_proxy_async_smem();
                    arrive(kv ? s_v_full[it & 1] : s_k_full[it & 1]);
                }
                arrive(s_code_empty[it & 1]);
            }
        }
    }
    if (warp >= 14) {
        // rows past a sequence's count are 0
        for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
            const int n = a.counts ? max(0, min(a.counts[b], a.tokens)) : a.tokens;
            const int64_t width = (int64_t)a.heads * D;
            float4* o = reinterpret_cast<float4*>(a.out + ((int64_t)b * a.tokens + n) * width);
            for (int64_t i = tid - 448; i < (a.tokens - n) * (width / 4); i += 64) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    // a wait that ran out (recorded): give what is in flight time to end before the memory goes
    if (s_abort)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int D>
int launch(const CacheAttArgs& a, cudaStream_t s) {
    static std::atomic<int> attr_set[64];
    int dev = 0;
    KZ_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        KZ_CHECK_CUDA(cudaFuncSetAttribute(cache_attention_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           Tc<D>::SMEM));
        if (dev >= 0 && dev < 64) attr_set[dev] = 1;
    }
    KZ_CHECK_CUDA(launch_pdl(cache_attention_tc_kernel<D>, dim3(a.ctas), dim3(kTcThreads), Tc<D>::SMEM, s, a));
    return KZ_OK;
}

}  // namespace

int launch_cache_attention_tc(const CacheAttArgs& a, int d, cudaStream_t s) {
    return d == 32 ? launch<32>(a, s) : d == 64 ? launch<64>(a, s) : launch<128>(a, s);
}

}  // namespace kz
