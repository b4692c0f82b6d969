// Attention over the paged int8 K/V cache: single tokens, chunks of a prompt,
// trees of drafted tokens.
//
//   s_l = (q . c_l) * ks_l * scale        c_l, ks_l: key l's codes and scale
//   o   = sum_l w_l * (vs_l * cv_l),  w = softmax(s) over the visible keys
//
// The new tokens' own K/V are in the cache already (positions length ..
// length + count - 1).  New token t sees every token before the new ones, and
// of the new ones its ancestors and itself in the tree (parents) or, without
// a tree, every one up to itself.  Rows past a sequence's count are 0.
//
// Arithmetic.  An int8 code is exact in fp16, so both products run on the
// tensor cores with the codes as they are, and the fp32 operand (q, and the
// weights times vs) as the sum of two fp16 values, which keeps 22 bits of it:
// q is scaled by a power of two per row so that its largest value lies in
// [2^13, 2^14), and the softmax's exponent is measured from the row's running
// maximum of s + log2(vs), which puts its largest w * vs there too, so that no
// half is lost to fp16's range (what is below 2^-38 of a row's largest is).
// Sums are 32-bit; the tensor core's sum of a step of keys is added to the row's
// sum by an fp32 multiply-add that also carries the softmax's rescaling, so that
// long contexts do not add up its truncation.  The small halves' products are
// summed first, or on their own, where the truncation costs least: 0.6e-6 of the
// output's size instead of 1.1e-6 at 8000 keys.
//
// Work.  The rows of one key head (its `group` query heads times the new
// tokens) form tiles of RT rows.  S^T = K Q^T and O^T = V^T P^T put the keys
// (the head's width) on the 16-row side of the mma and the query rows on its
// 8-column side, so that 8 rows, not 16, are the smallest tile and each code
// is converted once for all of a warp's rows.  Up to four rows leave half of
// those columns to the small halves (`halves in the columns`).  The four warps of a CTA split
// the keys of a tile (KG ways) and the rows (RG ways); each keeps its own
// running maximum and sum, joined at the end.  A fifth warp streams the pages
// by TMA (swizzled over the row, so ldmatrix reads without conflicts) into a
// ring of tiles of 128 keys.
//
// The keys of all sequences are cut into equal ranges, one per CTA, two CTAs
// a SM, so that ragged batches and long single sequences fill the GPU alike; a
// (sequence, head, row tile) that spans several ranges leaves its parts in the
// workspace, and a second kernel joins them.  Where that costs more than it
// gives (whole_ranges) each CTA takes whole row tiles instead.
//
// Measured, join included: 32 sequences of 4096 to 8191 keys, 32 heads over 8 key
// heads of 128, one new token each (416 MB of cache): 73 us = 5.7 TB/s, 0.87 of a
// plain copy; HBM bounds it but for about 7 us at the start and the join.  32
// sequences of up to 255 keys, 4 heads of 64: 7.2 us, latency (lengths, table,
// page, one after another, then a tile's chain).  One sequence of 30000: 23 us.
#include <algorithm>
#include <atomic>

#include "kz_cache_attention.cuh"

namespace kz {
namespace {

constexpr int kConsumers = 128;             // four warps compute, a fifth loads
constexpr int kCaThreads = kConsumers + 32;

// NT_ = 0: tiles of four rows, see `halves in the columns`.
template <int D, int NT_, int RG_>
struct Shape {
    static constexpr bool FOUR = NT_ == 0;
    static constexpr int NT = FOUR ? 1 : NT_, RG = RG_, KG = 4 / RG_;
    static constexpr int RT = FOUR ? 4 : 8 * NT * RG;       // rows a tile
    static constexpr int STEPS = kKT / (32 * KG);           // steps of 32 keys a warp takes in a tile
    static constexpr int STAGES = RT <= 16 ? 3 : 2;
    static constexpr int CODES = kKT * D, STAGE = 2 * CODES + 2 * kKT * 4;
    static constexpr int PITCH = D + 4;                     // joined rows: float2 stores without conflicts
    static constexpr int QBYTES = RT * D * 4;               // both halves of q, as mma operands
    static constexpr int UBYTES = RT * PITCH * 4 > QBYTES ? RT * PITCH * 4 : QBYTES;
    static constexpr int SMEM = STAGES * STAGE + UBYTES + 1024;
    static constexpr int SLOT = RT * (D + 2);               // floats of a part
};

// ------------------------------------------------------------ mma and codes

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <int D>
__device__ __forceinline__ uint32_t swizzled(uint32_t off) {   // byte offset in a tile of rows of D bytes
    return D == 128 ? off ^ ((off >> 3) & 0x70u) : D == 64 ? off ^ ((off >> 3) & 0x30u) : off ^ ((off >> 3) & 0x10u);
}

// 32 bytes of 16 keys (ldmatrix's order) as the 16-row operands of two mmas: of
// K with the keys on the rows, of V (transposed) with the head's width there,
// row x being d 2x and row x + 8 d 2x + 1.
struct Words {
    uint32_t r[4];
};
__device__ __forceinline__ Words ldsm4_of(uint32_t addr) {
    Words w;
    ldsm4(addr, w.r);
    return w;
}
__device__ __forceinline__ Words ldsm4_trans_of(uint32_t addr) {
    Words w;
    ldsm4_trans(addr, w.r);
    return w;
}
__device__ __forceinline__ void key_operands(Words w, uint32_t (&ops)[2][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w.r[j] ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ops[i][0] = two_codes<0x4140>(w.r[2 * i]);
        ops[i][1] = two_codes<0x4140>(w.r[2 * i + 1]);
        ops[i][2] = two_codes<0x4342>(w.r[2 * i]);
        ops[i][3] = two_codes<0x4342>(w.r[2 * i + 1]);
    }
}
__device__ __forceinline__ void value_operands(Words w, uint32_t (&ops)[2][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w.r[j] ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ops[i][0] = two_codes<0x4240>(w.r[2 * i]);
        ops[i][1] = two_codes<0x4341>(w.r[2 * i]);
        ops[i][2] = two_codes<0x4240>(w.r[2 * i + 1]);
        ops[i][3] = two_codes<0x4341>(w.r[2 * i + 1]);
    }
}

// ------------------------------------------------------------- the kernel

template <int D, int NT_, int RG>
__global__ void __launch_bounds__(kCaThreads, 2)
    cache_attention_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const CacheAttArgs a) {
    using S = Shape<D, NT_, RG>;
    constexpr int NT = S::NT;
    extern __shared__ uint8_t ca_smem[];
    uint8_t* ring = ca_smem + (-smem_u32(ca_smem) & 1023u);      // an offset, so that accesses stay shared-memory ones
    uint4* q_ops = reinterpret_cast<uint4*>(ring + S::STAGES * S::STAGE);   // [RT / 8][D / 16][32]: hi, hi, lo, lo
    float* joined = reinterpret_cast<float*>(q_ops);                        // [RT][PITCH], once q is done with
    __shared__ __align__(8) uint64_t s_full[S::STAGES], s_empty[S::STAGES];
    __shared__ uint32_t s_bad[S::STAGES];          // pages of a tile that are not there
    __shared__ float s_qs[S::RT];                  // a row's score factor
    __shared__ float s_m[S::KG][S::RT], s_l[S::KG][S::RT];
    __shared__ uint32_t s_sees[S::RT + 1][kTreeWords];
    __shared__ int32_t s_parent[KZ_TREE_MAX_NODES];
    __shared__ RangeShared s_range;
    __shared__ int s_abort;

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // uniform: so are the roles' branches
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 4);
        }
        s_abort = 0;
        fence_mbarrier_init();
    }
    griddep_wait();
    griddep_launch_dependents();

    if (warp < 4) find_range<S::RT>(a, s_range);
    __syncthreads();
    Walk<S::RT> walk(a, s_range.range);
    Segment g;
    int it = 0;      // tiles loaded or used so far

    if (warp == 4) {
        // ---- the loader: a lane a page of the tile
        const int pages = kKT >> a.c.shift;
        while (walk.next(a, g)) {
            const int held = g.len + g.count;                         // keys of the sequence
            auto page_id = [&](int t) {
                const int64_t pos = (int64_t)t * kKT + ((int64_t)lane << a.c.shift);
                return lane < pages && t < g.t1 && pos < held ? page_of(a.c, a.s, g.b, pos) : -2;   // -2: none needed
            };
            int id = page_id(g.t0);
            for (int t = g.t0; t < g.t1; ++t, ++it) {
                const int stage = it % S::STAGES;
                const int next = page_id(t + 1);
                mbar_wait(smem_u32(&s_empty[stage]), ((it / S::STAGES) & 1) ^ 1, a.status, &s_abort);
                const uint32_t there = __ballot_sync(0xffffffffu, id >= 0), bad = __ballot_sync(0xffffffffu, id == -1);
                const uint32_t full = smem_u32(&s_full[stage]);
                if (lane == 0) {
                    s_bad[stage] = bad;
                    if (bad) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
                    mbar_arrive_expect_tx(full, __popc(there) * a.c.page * (2 * D + 8));
                }
                __syncwarp();
                if (id >= 0) {
                    const uint32_t at = smem_u32(ring + stage * S::STAGE);
                    const int row = (id * a.c.heads + g.h) << a.c.shift, k0 = lane << a.c.shift;
                    tma_load_2d(at + k0 * D, &tm_k, full, 0, row);
                    tma_load_2d(at + S::CODES + k0 * D, &tm_v, full, 0, row);
                    bulk_load(at + 2 * S::CODES + k0 * 4, a.c.scale[0] + row, a.c.page * 4, full);
                    bulk_load(at + 2 * S::CODES + kKT * 4 + k0 * 4, a.c.scale[1] + row, a.c.page * 4, full);
                }
                id = next;
            }
        }
    } else {
        const int kg = warp / RG, rg = warp % RG, gq = lane >> 2, tq = lane & 3;
        // rows past a sequence's count are 0
        for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
            const int n = a.counts ? max(0, min(a.counts[b], a.tokens)) : a.tokens;
            const int64_t row = (int64_t)a.heads * D;
            float4* o = reinterpret_cast<float4*>(a.out + ((int64_t)b * a.tokens + n) * row);
            for (int64_t i = tid; i < (a.tokens - n) * (row / 4); i += kConsumers) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        bool first_segment = true;
        while (walk.next(a, g)) {
            const int rows = min(S::RT, g.count * a.group - g.rt * S::RT);   // of this tile
            // ---- q, both halves, as mma operands: lane (gq, tq) of [row / 8][d / 16] holds row gq, d 4 tq .. 4 tq + 3
            for (int n8 = warp; n8 < (S::RT + 7) / 8; n8 += 4) {
                const int r = S::FOUR ? gq & 3 : n8 * 8 + gq, R = g.rt * S::RT + r;
                float4 x[D / 16];
                uint32_t m = 0;
                const float* src = a.q + g.b * a.q_bs + (int64_t)(R / a.group) * a.q_rs +
                                   ((int64_t)g.h * a.group + R % a.group) * D + 4 * tq;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    x[i] = r < rows ? *reinterpret_cast<const float4*>(src + 16 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
                    const float e[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t bits = __float_as_uint(e[j]) & 0x7FFFFFFFu;
                        if (bits < 0x7F800000u) m = max(m, bits);
                    }
                }
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int ex = max((int)(m >> 23), 14);          // the row's largest exponent
                const float up = pow2_field(267 - ex);           // into [2^13, 2^14)
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const float e[4] = {x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up};
                    float hi[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) hi[j] = leading(e[j]);
                    const uint4 both = make_uint4(half2_bits(hi[0], hi[1]), half2_bits(hi[2], hi[3]),
                                                  half2_bits(e[0] - hi[0], e[1] - hi[1]), half2_bits(e[2] - hi[2], e[3] - hi[3]));
                    if constexpr (S::FOUR)
                        reinterpret_cast<uint2*>(q_ops)[i * 32 + lane] = gq < 4 ? make_uint2(both.x, both.y) : make_uint2(both.z, both.w);
                    else
                        q_ops[(n8 * (D / 16) + i) * 32 + lane] = both;
                }
                if (tq == 0 && (!S::FOUR || gq < 4)) s_qs[r] = a.scale * 1.4426950408889634f * pow2_field(ex - 13);   // scores in powers of 2
            }
            if (a.parents) {
                // each token's row of the tree: itself and its ancestors, one bit a node
                for (int j = tid; j <= g.last_token; j += kConsumers) s_parent[j] = a.parents[g.b * a.parents_bs + j];
                asm volatile("bar.sync 1, 128;" ::: "memory");
                for (int j = tid; j <= g.last_token - g.first_token; j += kConsumers) {
#pragma unroll
                    for (int w = 0; w < kTreeWords; ++w) s_sees[j][w] = 0;
                    for (int n = g.first_token + j; n >= 0;) {
                        s_sees[j][n >> 5] |= 1u << (n & 31);
                        const int up = s_parent[n];
                        n = up < n ? up : -1;
                    }
                }
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");

            float o[NT][D / 16][4], m[NT][2], l[NT][2], qs[NT][2];
            int token[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[n][i][j] = 0.0f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = S::FOUR ? 2 * (tq & 1) + j : (rg * NT + n) * 8 + 2 * tq + j;
                    m[n][j] = -INFINITY;
                    l[n][j] = 0.0f;
                    qs[n][j] = s_qs[r];
                    token[n][j] = (g.rt * S::RT + r) / a.group;
                }
            }
            const int limit = g.len + g.last_token + 1;           // keys that a row of the tile may see

            for (int t = g.t0; t < g.t1; ++t, ++it) {
                const int stage = it % S::STAGES;
                mbar_wait(smem_u32(&s_full[stage]), (it / S::STAGES) & 1, a.status, &s_abort);
                const uint32_t kt = smem_u32(ring + stage * S::STAGE), vt = kt + S::CODES;
                const float* ks_t = reinterpret_cast<const float*>(ring + stage * S::STAGE + 2 * S::CODES);
                const float* vs_t = ks_t + kKT;
                const uint32_t bad = s_bad[stage];
#pragma unroll 1
                for (int st = 0; st < S::STEPS; ++st) {
                    const int kl = (st * S::KG + kg) * 32, k0 = t * kKT + kl;   // first key, in the tile and the sequence
                    if (k0 >= limit) break;
                    const bool masked = k0 + 32 > g.len || bad;
                    // rows of 16 bytes for ldmatrix: keys (lane & 15), 16-byte column (lane >> 4)
                    const uint32_t row_at = (kl + (lane & 15)) * D + (lane >> 4) * 16;

                    if constexpr (S::FOUR) {
                        // ---- halves in the columns: four rows leave four of the mma's eight columns, which
                        // carry the small halves of q, then of the weights: half the mmas, and the lanes of
                        // either half take one 16 of the 32 keys each through the softmax
                        const bool upper = tq >= 2;                  // this lane's keys are the second 16
                        float s[2][4];
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                            for (int j = 0; j < 4; ++j) s[mt][j] = 0.0f;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt) {
                                uint32_t ops[2][4];
                                key_operands(ldsm4_of(kt + swizzled<D>(row_at + mt * 16 * D + c * 32)), ops);
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const uint2 q = reinterpret_cast<const uint2*>(q_ops)[(2 * c + i) * 32 + lane];
                                    mma_16816(s[mt], ops[i], q.x, q.y);
                                }
                            }
                        }
                        const int key0 = kl + (upper ? 16 : 0) + gq;
                        float z[4], mx[2] = {m[0][0], m[0][1]}, vs[2];
                        uint32_t seen = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + (e >> 1) * 8, tok = token[0][e & 1], j = t * kKT + key - g.len;
                            bool v = true;
                            if (masked) {
                                v = !((bad >> (key >> a.c.shift)) & 1u);
                                if (j >= 0)
                                    v = v && j < g.count && (a.parents ? tok <= g.last_token && ((s_sees[tok - g.first_token][j >> 5] >> (j & 31)) & 1u)
                                                                       : j <= tok);
                            }
                            seen |= (uint32_t)v << e;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float other = __shfl_xor_sync(0xffffffffu, upper ? s[0][e] : s[1][e], 2);
                            const float ks = ks_t[key0 + (e >> 1) * 8];
                            vs[e >> 1] = vs_t[key0 + (e >> 1) * 8];
                            z[e] = ((upper ? s[1][e] : s[0][e]) + other) * ks * qs[0][e & 1];
                            float x = z[e] + log2_vs(vs[e >> 1]);
                            if (!((seen >> e) & 1u)) z[e] = x = -INFINITY;
                            mx[e & 1] = fmaxf(mx[e & 1], x);
                        }
                        float corr[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int x = 2; x <= 16; x <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], x));
                            corr[j] = shrink(m[0][j], mx[j]);
                            m[0][j] = mx[j];
                            l[0][j] *= corr[j];
                            mx[j] = mx[j] == -INFINITY ? 0.0f : kLift - mx[j];
                        }
                        float hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float p = exp2_approx(z[e] + mx[e & 1]);
                            l[0][e & 1] = fmaf(p, kSumUnit, l[0][e & 1]);
                            const float w = (seen >> e) & 1u ? p * vs[e >> 1] : 0.0f;
                            hi[e] = leading(w);
                            lo[e] = w - hi[e];
                        }
                        uint32_t w[2][2];                            // [16 keys][8 keys]
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t h = half2_bits(hi[2 * j], hi[2 * j + 1]), k = half2_bits(lo[2 * j], lo[2 * j + 1]);
                            const uint32_t other = __shfl_xor_sync(0xffffffffu, upper ? h : k, 2);
                            w[0][j] = transposed_8x8(upper ? other : h);
                            w[1][j] = transposed_8x8(upper ? k : other);
                        }
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            float acc[2][4];
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt) {
                                uint32_t ops[2][4];
                                value_operands(ldsm4_trans_of(vt + swizzled<D>(row_at + mt * 16 * D + c * 32)), ops);
#pragma unroll
                                for (int i = 0; i < 2; ++i) mma_16816(acc[i], ops[i], w[mt][0], w[mt][1]);
                            }
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int j = 0; j < 4; ++j) o[0][2 * c + i][j] = fmaf(o[0][2 * c + i][j], corr[j & 1], acc[i][j]);
                        }
                        continue;
                    } else {
                        // ---- S^T: 32 keys x 8 NT rows
                        float s[2][NT][4], s_lo[2][NT][4];           // the small halves' products have a sum of their own
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[mt][n][j] = s_lo[mt][n][j] = 0.0f;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t ops[2][2][4];
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt) key_operands(ldsm4_of(kt + swizzled<D>(row_at + mt * 16 * D + c * 32)), ops[mt]);
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    const uint4 b = q_ops[((rg * NT + n) * (D / 16) + 2 * c + i) * 32 + lane];
#pragma unroll
                                    for (int mt = 0; mt < 2; ++mt) mma_16816(s[mt][n], ops[mt][i], b.x, b.y);
#pragma unroll
                                    for (int mt = 0; mt < 2; ++mt) mma_16816(s_lo[mt][n], ops[mt][i], b.z, b.w);
                                }
                        }

                        // ---- scales
                        float ks[2][2], vs[2][2], lv[2][2];
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                ks[mt][j] = ks_t[kl + mt * 16 + j * 8 + gq];
                                vs[mt][j] = vs_t[kl + mt * 16 + j * 8 + gq];
                                lv[mt][j] = log2_vs(vs[mt][j]);
                            }

                        // ---- softmax, one pass: new maximum, weights, and the weights times vs as two halves
                        float corr[NT][2];
                        uint32_t w_hi[2][NT][2], w_lo[2][NT][2];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            uint32_t seen = 0xFFu;          // bit 4 mt + 2 half + column
                            if (masked) {
                                seen = 0;
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const int key = kl + (e >> 2) * 16 + ((e >> 1) & 1) * 8 + gq, tok = token[n][e & 1];
                                    const int j = t * kKT + key - g.len;
                                    bool v = !((bad >> (key >> a.c.shift)) & 1u);
                                    if (j >= 0)
                                        v = v && j < g.count && (a.parents ? tok <= g.last_token && ((s_sees[tok - g.first_token][j >> 5] >> (j & 31)) & 1u)
                                                                           : j <= tok);
                                    seen |= (uint32_t)v << e;
                                }
                            }
                            float z[2][4];
                            float mx[2] = {m[n][0], m[n][1]};
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    z[mt][e] = (s[mt][n][e] + s_lo[mt][n][e]) * ks[mt][e >> 1] * qs[n][e & 1];
                                    float x = z[mt][e] + lv[mt][e >> 1];
                                    if (!((seen >> (4 * mt + e)) & 1u)) z[mt][e] = x = -INFINITY;
                                    mx[e & 1] = fmaxf(mx[e & 1], x);
                                }
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
#pragma unroll
                                for (int x = 4; x <= 16; x <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], x));
                                corr[n][j] = shrink(m[n][j], mx[j]);
                                m[n][j] = mx[j];
                                l[n][j] *= corr[n][j];
                                mx[j] = mx[j] == -INFINITY ? 0.0f : kLift - mx[j];      // -inf: no key yet, every weight is 0
                            }
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt) {
                                float hi[4], lo[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float p = exp2_approx(z[mt][e] + mx[e & 1]);
                                    l[n][e & 1] = fmaf(p, kSumUnit, l[n][e & 1]);
                                    const float w = (seen >> (4 * mt + e)) & 1u ? p * vs[mt][e >> 1] : 0.0f;
                                    hi[e] = leading(w);
                                    lo[e] = w - hi[e];
                                }
#pragma unroll
                                for (int j = 0; j < 2; ++j) {   // keys on the mma's inner side: transposed 8 x 8
                                    w_hi[mt][n][j] = transposed_8x8(half2_bits(hi[2 * j], hi[2 * j + 1]));
                                    w_lo[mt][n][j] = transposed_8x8(half2_bits(lo[2 * j], lo[2 * j + 1]));
                                }
                            }
                        }

                        // ---- O^T: D x 8 NT rows, the step's sum joined to the row's
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t ops[2][2][4];
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt) value_operands(ldsm4_trans_of(vt + swizzled<D>(row_at + mt * 16 * D + c * 32)), ops[mt]);
                            float acc[2][NT][4];
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt)             // the small halves first: their sum is truncated least
#pragma unroll
                                for (int i = 0; i < 2; ++i)
#pragma unroll
                                    for (int n = 0; n < NT; ++n) mma_16816(acc[i][n], ops[mt][i], w_lo[mt][n][0], w_lo[mt][n][1]);
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
#pragma unroll
                                    for (int n = 0; n < NT; ++n) mma_16816(acc[i][n], ops[mt][i], w_hi[mt][n][0], w_hi[mt][n][1]);
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        o[n][2 * c + i][j] = fmaf(o[n][2 * c + i][j], corr[n][j & 1], acc[i][n][j]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_empty[stage]));
            }

            // ---- the warps' parts joined
            if constexpr (S::FOUR) {                               // the small halves' sums to the leading ones'
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[0][i][j] += __shfl_xor_sync(0xffffffffu, o[0][i][j], 2);
            }
            const bool holds = !S::FOUR || tq < 2;                 // a lane whose rows are not another's too
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int x = S::FOUR ? 2 : 4; x <= 16; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
                    if (gq == 0 && holds) {
                        s_m[kg][(rg * NT + n) * 8 + 2 * tq + j] = m[n][j];
                        s_l[kg][(rg * NT + n) * 8 + 2 * tq + j] = l[n][j];
                    }
                }
            asm volatile("bar.sync 1, 128;" ::: "memory");     // and q is done with
            const bool direct = g.whole;
            float* slot = direct ? nullptr : a.parts + (2 * (int64_t)blockIdx.x + (first_segment ? 0 : 1)) * S::SLOT;
            first_segment = false;
            float* out = a.out + (int64_t)g.b * a.tokens * a.heads * D + (int64_t)g.h * a.group * D;
            auto out_row = [&](int r) {                         // row r of the tile in `out`
                const int R = g.rt * S::RT + r;
                return out + ((int64_t)(R / a.group) * a.heads + R % a.group) * D;
            };
            for (int turn = 0; turn < S::KG; ++turn) {
                if (turn == kg && holds) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int r = (rg * NT + n) * 8 + 2 * tq + j;
                            float M = -INFINITY;
#pragma unroll
                            for (int k = 0; k < S::KG; ++k) M = fmaxf(M, s_m[k][r]);
                            const float f = shrink(m[n][j], M);
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                float2* p = reinterpret_cast<float2*>(joined + r * S::PITCH + 16 * i + 2 * gq);
                                const float2 v = turn ? *p : make_float2(0.f, 0.f);
                                *p = make_float2(fmaf(o[n][i][j], f, v.x), fmaf(o[n][i][j + 2], f, v.y));
                            }
                        }
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
            for (int i = tid; i < rows * (D / 4); i += kConsumers) {
                const int r = i / (D / 4), c = i % (D / 4);
                float4 v = *reinterpret_cast<const float4*>(joined + r * S::PITCH + 4 * c);
                if (direct) {
                    float M = -INFINITY, L = 0.0f;
#pragma unroll
                    for (int k = 0; k < S::KG; ++k) M = fmaxf(M, s_m[k][r]);
#pragma unroll
                    for (int k = 0; k < S::KG; ++k) L += s_l[k][r] * shrink(s_m[k][r], M);
                    const float f = L == 0.0f ? 0.0f : 1.0f / L;
                    v = make_float4(over_sum(v.x, f), over_sum(v.y, f), over_sum(v.z, f), over_sum(v.w, f));
                }
                *reinterpret_cast<float4*>((direct ? out_row(r) : slot + r * D) + 4 * c) = v;
            }
            if (!direct && tid < S::RT) {
                float M = -INFINITY, L = 0.0f;
                for (int k = 0; k < S::KG; ++k) M = fmaxf(M, s_m[k][tid]);
                for (int k = 0; k < S::KG; ++k) L += s_l[k][tid] * shrink(s_m[k][tid], M);
                slot[S::RT * D + tid] = M;
                slot[S::RT * D + S::RT + tid] = L;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");     // q, maxima and the joined rows are free again
        }
    }
    __syncthreads();
    // a wait that ran out (recorded): give the copies in flight time to land before the shared memory goes
    if (s_abort)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

// Joins the parts of a (sequence, head, row tile) that several CTAs left: with
// M the largest of their maxima, o = sum f_c o_c / sum f_c l_c, f_c =
// 2^(m_c - M).  Latency bounds it (a row's parts are far apart), so a lane has D /
// 32 neighbouring values of a row, one load each.  FEW: up to four parts are a
// warp's work, every load of two rows in flight at once, and a block has eight
// rows and four warps.  Otherwise (more CTAs than four a row tile: few, long
// sequences) a block has one row, dealt out part by part to eight warps, each
// with a maximum of its own, and joined once more.  The attention with the first
// and the second: one sequence of 30000 keys (35 parts a row) 31 and 23 us; 32
// sequences of 4096 to 8191 76 and 80; 2 chunks of 500 tokens, 4 rows a token, 150
// and 188.
template <bool FEW, int RT>
struct Join {
    static constexpr int ROWS = !FEW ? 1 : RT < 8 ? RT : 8, WARPS = FEW ? 4 : 8;
};
template <int E>
__device__ __forceinline__ void load_values(const float* p, float (&v)[E]) {
    if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else if constexpr (E == 2) {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] = x.x, v[1] = x.y;
    } else {
        v[0] = *p;
    }
}
template <int E>
__device__ __forceinline__ void store_values(float* p, const float (&v)[E]) {
    if constexpr (E == 4)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (E == 2)
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    else
        *p = v[0];
}
template <int D, int RT, bool FEW>
__global__ void __launch_bounds__(32 * Join<FEW, RT>::WARPS) cache_attention_join_kernel(const CacheAttArgs a) {
    constexpr int E = D / 32, SLOT = RT * (D + 2), ROWS = Join<FEW, RT>::ROWS, WARPS = Join<FEW, RT>::WARPS, BLOCKS = RT / ROWS;
    __shared__ Work s_work[WARPS];
    __shared__ int s_before[WARPS];
    __shared__ __align__(16) float s_part[WARPS][ROWS][D];
    __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS];
    griddep_launch_dependents();
    const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // lengths and counts were written before the kernel that left the parts began
    Work w{0, 0, 0};
    int before = 0;
    for (int i = threadIdx.x; i < a.batch; i += 32 * WARPS) {
        const Seq s = sequence<RT>(a, i);
        w.add(a, s);
        if (i < b) before += units_of(a, s, false);
    }
    w.add_warp();
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) {
        s_work[warp] = w;
        s_before[warp] = before;
    }
    __syncthreads();
    w = s_work[0];
    before = s_before[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) {
        w.add(s_work[i]);
        before += s_before[i];
    }
    const Seq s = sequence<RT>(a, b);
    const int tile = blockIdx.x / BLOCKS, h = tile % a.c.heads, rt = tile / a.c.heads;
    const int r0 = (blockIdx.x % BLOCKS) * ROWS, rows = min(RT, s.count * a.group - rt * RT) - r0;   // of this block
    const int per = max(1, a_cta(a, w.units));
    const int u0 = before + (h * s.row_tiles + rt) * s.tiles, c0 = u0 / per, c1 = (u0 + s.tiles - 1) / per;
    griddep_wait();
    if (whole_ranges(a, w) || rt >= s.row_tiles || rows <= 0 || c0 == c1) return;     // nothing, or one CTA had it all
    auto slot = [&](int c) {                                    // a CTA's first part is in its first slot
        return a.parts + (2 * (int64_t)c + (c > c0 || c0 * per == u0 ? 0 : 1)) * SLOT;
    };
    auto finish = [&](int r, float L, float (&o)[E]) {
        const float f = L == 0.0f ? 0.0f : 1.0f / L;
        const int R = rt * RT + r;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = over_sum(o[e], f);
        store_values(a.out + ((int64_t)b * a.tokens + R / a.group) * a.heads * D + ((int64_t)h * a.group + R % a.group) * D + lane * E, o);
    };
    if (c1 - c0 < 4) {
        for (int i = warp; i < min(rows, ROWS); i += 2 * WARPS) {
            float m[2][4], l[2][4], v[2][4][E];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int r = r0 + i + k * WARPS;
                    const bool there = c <= c1 - c0 && i + k * WARPS < min(rows, ROWS);
                    const float* p = slot(there ? c0 + c : c0);
                    m[k][c] = there ? p[RT * D + r] : -INFINITY;
                    l[k][c] = there ? p[RT * D + RT + r] : 0.0f;
                    if (there) load_values(p + r * D + lane * E, v[k][c]);
                }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (i + k * WARPS >= min(rows, ROWS)) break;
                const float M = fmaxf(fmaxf(m[k][0], m[k][1]), fmaxf(m[k][2], m[k][3]));
                float L = 0.0f, o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c > c1 - c0) break;
                    const float f = shrink(m[k][c], M);
                    L = fmaf(l[k][c], f, L);
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = fmaf(v[k][c][e], f, o[e]);
                }
                finish(r0 + i + k * WARPS, L, o);
            }
        }
        return;
    }
    for (int i = 0; i < min(rows, ROWS); ++i) {
        // a warp's parts: c0 + warp, c0 + warp + WARPS, ...
        const int r = r0 + i;
        float M = -INFINITY, L = 0.0f, o[E];
        for (int c = c0 + warp + WARPS * lane; c <= c1; c += 32 * WARPS) M = fmaxf(M, slot(c)[RT * D + r]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll 8
        for (int c = c0 + warp; c <= c1; c += WARPS) {
            const float* p = slot(c);
            const float f = shrink(p[RT * D + r], M);
            L = fmaf(p[RT * D + RT + r], f, L);
            float v[E];
            load_values(p + r * D + lane * E, v);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], f, o[e]);
        }
        store_values(&s_part[warp][i][lane * E], o);
        if (lane == 0) {
            s_m[warp][i] = M;
            s_l[warp][i] = L;
        }
    }
    __syncthreads();
    for (int i = warp; i < min(rows, ROWS); i += WARPS) {
        float M = -INFINITY, L = 0.0f, o[E];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][i]);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = shrink(s_m[w][i], M);
            L = fmaf(s_l[w][i], f, L);
            float v[E];
            load_values(&s_part[w][i][lane * E], v);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], f, o[e]);
        }
        finish(r0 + i, L, o);
    }
}

template <int D, int RT, bool FEW>
int launch_join_as(const CacheAttArgs& a, int64_t row_tiles, cudaStream_t s) {
    using J = Join<FEW, RT>;
    KZ_CHECK_CUDA(launch_pdl(cache_attention_join_kernel<D, RT, FEW>,
                             dim3((unsigned)(row_tiles * a.c.heads * (RT / J::ROWS)), (unsigned)a.batch), dim3(32 * J::WARPS),
                             0, s, a));
    return KZ_OK;
}
template <int D, int RT>
int launch_join(const CacheAttArgs& a, int64_t row_tiles, cudaStream_t s) {
    return a.ctas <= 4 * (int64_t)a.batch * a.c.heads * row_tiles ? launch_join_as<D, RT, true>(a, row_tiles, s)
                                                       : launch_join_as<D, RT, false>(a, row_tiles, s);
}

// ---------------------------------------------------------------- launches

// Rows of a tile: the smallest of 4, 8, 16 and 32 that holds a key head's rows.  With
// tiles of 4, 8, 16 and 32, 4 rows over 32 long sequences: 73, 76, 110 and 197 us
// (4 and 8 for seconds on end, under the power cap: 79 and 86); 16 rows, 16
// sequences of 3000 to 6000: 51 us with 16, 84 with 32 (which spills 152 bytes a
// thread at heads of 128).
int tile_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }

// Whether a call needs no workspace and no join: its table holds no more than
// four tiles of keys a row tile.  One sequence of 500 keys, 8 key heads: 8.6 us so,
// 9.0 in ranges; 8 sequences 9.2 and 10.9; 32 11.8 and 16.2.
bool short_table(int64_t cols, int64_t page) { return cols * page <= 4 * kKT; }

// Whether the rows of a key head are many enough for the tcgen05 kernel, whose
// time does not depend on them up to 128: at 32 rows (batch 16, 8 key heads of
// 128, contexts of 1500 and 6000) it takes 36.6 and 85.6 us against 36.8 and 86.2
// here, with heads of 64 (20 rows, 32 contexts of 5000) 124 against 87; at 64
// rows of heads of 128 51 and 98 against 58 and 150 with tiles of 64 rows.  Both at
// each width, 16 contexts of up to 6000, 4 key heads (there, here): of 128 20 rows
// 49.6, 54.4, 32 50.2, 55.8, 36 50.3, 67.8, 64 53.8, 87.7 us; of 64 44.2, 36.8, 44.4,
// 37.7, 44.3, 47.0, 45.3, 55.9; of 32 37.3, 29.9, 37.7, 30.7, 37.6, 39.1, 38.5, 44.2.
// Of up to 300 the other way round for 36 to 64 rows: of 64 12.2 and 10.8, of 32 11.2
// and 9.0 us, which one rule for all lengths costs.
bool many_rows(int64_t rows) { return rows > 32; }

int64_t tile_of(int64_t rows) { return many_rows(rows) ? kTcRows : tile_rows(rows); }
int64_t row_tiles_of(int64_t rows) { return (rows + tile_of(rows) - 1) / tile_of(rows); }

int64_t parts_floats(int64_t rows, int64_t d) {
    const int64_t ctas = (many_rows(rows) ? 1 : 2) * (int64_t)sm_count();
    return 2 * ctas * tile_of(rows) * (d + 2);
}

template <int D, int NT, int RG>
int launch_cache_attention(CacheAttArgs a, int64_t row_tiles, cudaStream_t s) {
    using S = Shape<D, NT, RG>;
    static std::atomic<int> attr_set[64];
    int dev = 0;
    KZ_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        KZ_CHECK_CUDA(cudaFuncSetAttribute(cache_attention_kernel<D, NT, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           S::SMEM));
        if (dev >= 0 && dev < 64) attr_set[dev] = 1;
    }
    CUtensorMap tm_k, tm_v;
    const uint64_t rows = (uint64_t)a.c.pages * a.c.heads * a.c.page;
    int st = tensor_map_rows_i8(&tm_k, a.c.codes[0], D, rows, (uint32_t)a.c.page);
    if (!st) st = tensor_map_rows_i8(&tm_v, a.c.codes[1], D, rows, (uint32_t)a.c.page);
    if (st) return st;
    const int64_t most = (int64_t)a.batch * a.c.heads * row_tiles;
    a.ctas = (int)std::min<int64_t>(2 * (int64_t)sm_count(), a.parts ? 2 * (int64_t)sm_count() : most);
    a.by_ctas = fast_div((uint32_t)a.ctas);
    KZ_CHECK_CUDA(launch_pdl(cache_attention_kernel<D, NT, RG>, dim3(a.ctas), dim3(kCaThreads), S::SMEM, s, tm_k, tm_v, a));
    return a.parts ? launch_join<D, S::RT>(a, row_tiles, s) : KZ_OK;
}

template <int D>
int dispatch_cache_attention(CacheAttArgs a, cudaStream_t s) {
    const int64_t rows = (int64_t)a.tokens * a.group, row_tiles = row_tiles_of(rows);
    if (many_rows(rows)) {
        a.ctas = (int)std::min<int64_t>(sm_count(), a.parts ? sm_count() : (int64_t)a.batch * a.c.heads * row_tiles);
        a.by_ctas = fast_div((uint32_t)a.ctas);
        const int st = launch_cache_attention_tc(a, D, s);
        return st || !a.parts ? st : launch_join<D, kTcRows>(a, row_tiles, s);
    }
    const int rt = tile_rows(rows);
    if (rt == 4) return launch_cache_attention<D, 0, 1>(a, row_tiles, s);
    if (rt == 8) return launch_cache_attention<D, 1, 1>(a, row_tiles, s);
    if (rt == 16) return launch_cache_attention<D, 2, 1>(a, row_tiles, s);
    return launch_cache_attention<D, 2, 2>(a, row_tiles, s);
}

}  // namespace
}  // namespace kz

using namespace kz;

extern "C" size_t kz_cache_attention_workspace_bytes(const kz_cache* cache, int64_t tokens, int64_t heads,
                                                     int64_t table_cols) {
    if (!cache || cache->kv_heads <= 0 || tokens <= 0 || heads <= 0 || table_cols < 0) return 0;
    if (short_table(table_cols, cache->page_size)) return 0;
    return sizeof(float) * (size_t)parts_floats(tokens * (heads / cache->kv_heads), cache->head_dim);
}

extern "C" int kz_cache_attention_f32(const kz_cache* cache, const float* q, int64_t batch, int64_t tokens,
                                      int64_t heads, int64_t q_batch_stride, int64_t q_row_stride,
                                      const int32_t* table, int64_t table_cols, const int32_t* lengths,
                                      const int32_t* counts, const int32_t* parents, int64_t parents_batch_stride,
                                      float scale, float* out, void* workspace, size_t workspace_bytes,
                                      kz_stream_t stream) {
    CacheAttArgs a;
    int st = cache_view(cache, "kz_cache_attention_f32", &a.c);
    if (!st) st = seq_view(table, table_cols, lengths, batch, "kz_cache_attention_f32", &a.s);
    if (st) return st;
    KZ_REQUIRE(heads > 0 && heads < (1 << 16) && heads % cache->kv_heads == 0,
               "kz_cache_attention_f32: heads must be a multiple of kv_heads");
    KZ_REQUIRE(batch < 65536, "kz_cache_attention_f32: batch must be below 65536");
    KZ_REQUIRE(tokens >= 0 && tokens < (1 << 24) && tokens * heads < (int64_t)INT32_MAX / 64,
               "kz_cache_attention_f32: tokens * heads out of range");
    KZ_REQUIRE(table_cols * cache->page_size < (int64_t)INT32_MAX - (1 << 25),
               "kz_cache_attention_f32: table_cols * page_size out of range");
    const int64_t most_tiles = (table_cols * cache->page_size + tokens) / kKT + 1;
    KZ_REQUIRE(batch * cache->kv_heads * row_tiles_of(tokens * (heads / cache->kv_heads)) < (int64_t)INT32_MAX / most_tiles,
               "kz_cache_attention_f32: the call's work is out of range");
    if (batch * tokens == 0) return KZ_OK;
    KZ_REQUIRE(q && out, "kz_cache_attention_f32: q or out is NULL");
    KZ_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0 &&
                   ((q_batch_stride | q_row_stride) & 3) == 0,
               "kz_cache_attention_f32: q and out must be 16-byte aligned, strides multiples of 4 floats");
    KZ_REQUIRE(q_batch_stride >= 0 && (tokens == 1 || q_row_stride >= heads * cache->head_dim),
               "kz_cache_attention_f32: q's row stride is shorter than heads * head_dim");
    KZ_REQUIRE(!parents || tokens <= KZ_TREE_MAX_NODES, "kz_cache_attention_f32: a tree has at most 256 nodes");
    KZ_REQUIRE(parents_batch_stride == 0 || parents_batch_stride >= tokens,
               "kz_cache_attention_f32: parents_batch_stride is shorter than tokens");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (cache->pages == 0) {   // no key anywhere
        st = check_device();
        if (st) return st;
        KZ_CHECK_CUDA(cudaMemsetAsync(out, 0, sizeof(float) * batch * tokens * heads * cache->head_dim, s));
        return KZ_OK;
    }
    const size_t need = kz_cache_attention_workspace_bytes(cache, tokens, heads, table_cols);
    KZ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0),
               "kz_cache_attention_f32: workspace too small or not 16-byte aligned");
    st = check_device();
    if (st) return st;
    a.q = q;
    a.q_bs = q_batch_stride;
    a.q_rs = q_row_stride;
    a.counts = counts;
    a.parents = parents;
    a.parents_bs = parents_batch_stride;
    a.out = out;
    a.parts = need ? static_cast<float*>(workspace) : nullptr;
    a.batch = (int)batch;
    a.tokens = (int)tokens;
    a.heads = (int)heads;
    a.group = (int)(heads / cache->kv_heads);
    a.scale = scale;
    a.status = device_status_ptr();
    return cache->head_dim == 32   ? dispatch_cache_attention<32>(a, s)
           : cache->head_dim == 64 ? dispatch_cache_attention<64>(a, s)
                                   : dispatch_cache_attention<128>(a, s);
}
