// Verification of a tree of drafted tokens against the target's probabilities
// (speculative sampling, children tried one after another), from given random
// numbers.
//
// With p[n] the target's row at node n, q[n] the draft's row the children of n
// were drawn from (one-hot at the child's token where there is no draft row),
// node 0 the root, r = p[0]:
//   for j = 1 .. N-1 in order, if parent[j] is the current node:
//     u[j] * q(x[j]) < r(x[j])   accept: j becomes the current node, r = p[j]
//     otherwise                  reject: r = (r - q)+ / sum (r - q)+  (unchanged where that sum is 0)
// and the next token is the smallest i with r(0) + .. + r(i) > u * sum r.
// A row that a decision takes a sum of and that is not finite is recorded in the
// status word; the sequence's answers then are some nodes and some token.
// Everything is computed in double from the fp32 rows (or in two fp32 parts
// that keep as much), so that the decisions do not depend on how the work is
// split.
//
// After k rejections at a node r is (p - c_k q)+ / t_k with c_0 = 0, t_0 = 1,
// c_(k+1) = c_k + t_k and t_(k+1) = sum (p - c_(k+1) q)+: dividing the rule's
// r_k = (p - c_k q)+ / t_k through, (r_k - q)+ is (p - (c_k + t_k) q)+ / t_k.
//
// Each sequence is walked by one cluster: every CTA takes a slice of the
// vocabulary and repeats the walk itself (the accept tests need single values
// only, gathered up front), so that the cluster meets once a rejection and
// once at the end, to exchange the slices' sums through distributed shared
// memory.  With a draft each rejection is a pass over two rows; if the walk
// ends with it, its sums are those that the last token is drawn by.  Without
// one r is p with the rejected tokens taken out, over what is left: one pass
// over a node's row gives its sum, from which each rejected token's p is
// subtracted.  Nothing else of the probabilities is touched.  What bounds it: for
// each rejection a pass, a meeting and the walk, one after another.  The passes
// of a whole batch run at the memory's rate (33 MB in 4.4 us, the first from HBM, the
// later ones from L2), on values that an earlier pass at the node had in registers
// already; meetings and walk (2 to 3 us) are latency.  A warp loads all of its
// part of a slice (8 chunks, 128 values of each at a time) before it adds anything
// up; two CTAs a SM leave 128 registers a thread for it, 44 bytes of which spill.
//
// Measured: 32 trees of 16 nodes over 128000 tokens with a draft, 26 to 28 us (32.8
// MB of rows once: 5 us); 32 trees of 6 nodes over 65 tokens, no draft: 10.5 us.
// Rows that do not start on 16 bytes are read by the word: 32 trees of 16 over 50257
// tokens 20.0 us, over 50256 16.0; without a draft 13.2 and 12.1.  Before the walk lost its divisions and the draw its serial sums (30 us) the
// first took 42 us with clusters of 4, 40 with blocks of 128 threads and 32 with
// every sum in double.
#include <math.h>

#include <algorithm>

#include "kz_common.cuh"

namespace kz {
namespace {

constexpr int kVThreads = 256, kVWarps = kVThreads / 32, kVChunks = 8;
constexpr int kVMaxNodes = 1024;
constexpr int kVMaxCluster = 8;

struct VerifyArgs {
    const int64_t* tokens;     // [B, N]
    const int32_t* parents;    // [B, N], or [N] with parents_bs 0
    int64_t parents_bs;
    const float* target;       // [B, N, V]
    const float* draft;        // [B, N, V] or NULL
    const float* accept_u;     // [B, N]
    const float* sample_u;     // [B]
    int32_t* path;             // [B, N]
    int32_t* count;            // [B]
    int64_t* next;             // [B]
    int nodes, vocab, chunk;   // chunk: a multiple of 128 values; a warp has kVChunks, a slice all its warps' chunks
    int wide;                  // rows start on 16 bytes
    int* status;
};

struct VerifyShared {
    double sum[2][kVMaxCluster];       // the slices' sums, a buffer for each of two successive meetings
    double chunk_sum[kVWarps][kVChunks];
    // the rejections at the current node
    double c, t;                       // see above; without a draft t is the sum of what is left
    double gone_p[kVMaxNodes];         // without a draft: the rejected tokens and their p
    int gone[kVMaxNodes];
    float p_at[kVMaxNodes], q_at[kVMaxNodes], u[kVMaxNodes];
    int parent[kVMaxNodes], token[kVMaxNodes];
    int rejections, node, child, found;
    int summed;                        // the node whose sums are in `sum` and `chunk_sum`: of p without a draft, with
                                       // one of (p - c q)+
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// x+, and NaN where x is: a row that is no distribution must not become one
__device__ __forceinline__ double rest_of(double x) { return x < 0.0 ? 0.0 : x; }
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ bool is_gone(const VerifyShared& s, int x) {
    for (int k = 0; k < s.rejections; ++k)
        if (s.gone[k] == x) return true;
    return false;
}
// whether node j is accepted, u q < r at its token, of its parent's row (t times it: no division)
__device__ __forceinline__ bool accepts(const VerifyShared& s, bool has_draft, int j) {
    const double p = s.p_at[j], q = s.q_at[j], rest = has_draft ? rest_of(p - s.c * q) : is_gone(s, s.token[j]) ? 0.0 : p;
    return (double)s.u[j] * q * s.t < rest;
}
// without a draft, the node's sum known: token of node j rejected
__device__ __forceinline__ void take_out(VerifyShared& s, int j, double sum) {
    if (is_gone(s, s.token[j])) return;
    const double left = (s.rejections == 0 ? sum : s.t) - (double)s.p_at[j];
    if (!(left > 0.0)) return;
    s.t = left;
    s.gone[s.rejections] = s.token[j];
    s.gone_p[s.rejections++] = s.p_at[j];
}

// Sums of eight values a lane over the warp: lane l gets value (l >> 2)'s in
// nine exchanges, each of the first three halving the values a lane has.
__device__ __forceinline__ double warp_sums_f64(double (&v)[kVChunks]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 4; h > 0; h >>= 1) {
        const bool up = lane & (4 * h);
#pragma unroll
        for (int i = 0; i < h; ++i) {
            const double give = up ? v[i] : v[i + h], keep = up ? v[i + h] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * h);
        }
    }
    double t = v[0];
    t += __shfl_xor_sync(0xffffffffu, t, 2);
    t += __shfl_xor_sync(0xffffffffu, t, 1);
    return t;
}

// Sums of fp32 values without a double per value (whose conversions and
// additions bound the pass): pairs of values added to a sum kept as two fp32
// parts, each addition's rounding error recovered (Knuth's two-sum) and kept in
// the second.  n additions lose at most n 2^-48 of the terms' sum.
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
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
struct TwoPart {
    uint64_t hi, lo;       // two sums side by side
    __device__ __forceinline__ void add(uint64_t x) {
        const uint64_t s = add2(hi, x), b = sub2(s, hi);
        lo = add2(lo, add2(sub2(hi, sub2(s, b)), sub2(x, b)));
        hi = s;
    }
    // adds (p - q)+ = p - min(p, q): the difference's own rounding error is exact, as p is the larger
    __device__ __forceinline__ void add_rest(float p0, float p1, float q0, float q1) {
        const uint64_t p = pair(p0, p1), q = pair(min_nan(q0, p0), min_nan(q1, p1)), d = sub2(p, q);
        add(d);
        lo = add2(lo, sub2(sub2(p, d), q));
    }
    __device__ __forceinline__ double sum() const {
        float a, b, c, d;
        unpair(hi, a, b);
        unpair(lo, c, d);
        return ((double)a + (double)b) + ((double)c + (double)d);
    }
};

// Four values of a row from i on, 0 at and past `end`.
__device__ __forceinline__ float4 four(const float* row, int i, int end, int wide) {
    if (wide && i + 3 < end) return __ldg(reinterpret_cast<const float4*>(row + i));
    return make_float4(i < end ? __ldg(row + i) : 0.0f, i + 1 < end ? __ldg(row + i + 1) : 0.0f,
                       i + 2 < end ? __ldg(row + i + 2) : 0.0f, i + 3 < end ? __ldg(row + i + 3) : 0.0f);
}

__global__ void __launch_bounds__(kVThreads, 2) verify_tree_kernel(VerifyArgs a) {
    __shared__ VerifyShared s;
    // every CTA of the cluster has begun before the first sum goes into another's shared memory
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
    const int64_t b = blockIdx.x / ranks;
    const float* target = a.target + b * a.nodes * (int64_t)a.vocab;
    const float* draft = a.draft ? a.draft + b * a.nodes * (int64_t)a.vocab : nullptr;
    for (int j = tid; j < a.nodes; j += blockDim.x) {
        const int parent = a.parents[b * a.parents_bs + j];
        const int64_t x = a.tokens[b * a.nodes + j];
        bool child = j > 0 && parent >= 0 && parent < j;
        if (child && (x < 0 || x >= a.vocab)) {   // no token: never accepted, rejects nothing
            record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
            child = false;
        }
        s.parent[j] = child ? parent : -1;
        s.token[j] = child ? (int)x : -1;
        s.u[j] = a.accept_u[b * a.nodes + j];
        s.p_at[j] = child ? target[parent * (int64_t)a.vocab + x] : 0.0f;
        s.q_at[j] = child && draft ? draft[parent * (int64_t)a.vocab + x] : 1.0f;
        if (rank == 0) a.path[b * a.nodes + j] = j == 0 ? 0 : -1;
    }
    if (tid == 0) {
        s.rejections = 0;
        s.node = 0;
        s.c = 0.0;
        s.t = 1.0;
        s.child = 1;
        s.found = -1;
        s.summed = -1;
    }
    const double sample_u = (double)a.sample_u[b];
    int accepted = 1, meeting = 0;
    // this warp's values [lo, end), chunk c at lo + c * chunk
    const int span = kVChunks * a.chunk;
    const int slice0 = (int)min((int64_t)a.vocab, (int64_t)rank * warps * span);
    const int lo = (int)min((int64_t)a.vocab, (int64_t)slice0 + (int64_t)warp * span);
    for (;;) {
        __syncthreads();
        if (tid == 0) {
            // walk to the next rejection (s.found: the rejected child) or past the last node
            s.found = -1;
            int j = s.child;
            for (; j < a.nodes; ++j) {
                if (s.parent[j] != s.node) continue;
                if (accepts(s, draft != nullptr, j)) {
                    s.node = j;
                    s.rejections = 0;
                    s.c = 0.0;
                    s.t = 1.0;
                    if (rank == 0) a.path[b * a.nodes + accepted] = j;
                    ++accepted;
                } else if (!draft && s.summed == s.node) {
                    double sum = 0.0;
                    for (int c = 0; c < (int)ranks; ++c) sum += s.sum[(meeting & 1) ^ 1][c];
                    take_out(s, j, sum);
                } else {
                    s.found = j;
                    break;
                }
            }
            s.child = j + 1;
        }
        __syncthreads();
        const int node = s.node, rejected = s.found;
        const float* p = target + node * (int64_t)a.vocab;
        const float* q = draft ? draft + node * (int64_t)a.vocab : nullptr;
        const bool known = rejected < 0 && s.summed == node;
        // what is summed: (p - c q)+, p where c is 0
        const double c_now = !q ? 0.0 : rejected >= 0 ? s.c + s.t : s.c;
        auto values = [&](const float4& pi, const float4& qi, double (&r)[4]) {
            const float pe[4] = {pi.x, pi.y, pi.z, pi.w}, qe[4] = {qi.x, qi.y, qi.z, qi.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = c_now == 0.0 ? (double)pe[e] : rest_of((double)pe[e] - c_now * (double)qe[e]);
        };
        double sum[kVChunks];
#pragma unroll
        for (int c = 0; c < kVChunks; ++c) sum[c] = 0.0;
        if (lo < a.vocab && !known) {
            TwoPart part[kVChunks];
#pragma unroll
            for (int c = 0; c < kVChunks; ++c) part[c] = {0, 0};
            for (int i0 = 4 * lane; i0 < a.chunk; i0 += 128) {
                float4 pv[kVChunks], qv[kVChunks];
#pragma unroll
                for (int c = 0; c < kVChunks; ++c) {
                    const int i = (int)min((int64_t)a.vocab, (int64_t)lo + (int64_t)c * a.chunk + i0);
                    pv[c] = four(p, i, a.vocab, a.wide);
                    qv[c] = c_now != 0.0 ? four(q, i, a.vocab, a.wide) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                if (c_now == 0.0) {
#pragma unroll
                    for (int c = 0; c < kVChunks; ++c) {
                        part[c].add(pair(pv[c].x, pv[c].y));
                        part[c].add(pair(pv[c].z, pv[c].w));
                    }
                } else if (c_now == 1.0) {         // the first rejection
#pragma unroll
                    for (int c = 0; c < kVChunks; ++c) {
                        part[c].add_rest(pv[c].x, pv[c].y, qv[c].x, qv[c].y);
                        part[c].add_rest(pv[c].z, pv[c].w, qv[c].z, qv[c].w);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kVChunks; ++c) {
                        double r[4];
                        values(pv[c], qv[c], r);
                        sum[c] += (r[0] + r[1]) + (r[2] + r[3]);
                    }
                }
            }
            if (c_now == 0.0 || c_now == 1.0) {
#pragma unroll
                for (int c = 0; c < kVChunks; ++c) sum[c] = part[c].sum();
            }
        }
        if (!known) {
            const double all = warp_sums_f64(sum);
            if ((lane & 3) == 0) s.chunk_sum[warp][lane >> 2] = all;
            __syncthreads();
            if (meeting == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // (the first turn always sums)
            if (warp == 0) {
                // the slice's sum, to every CTA of the cluster
                double t = 0.0;
                for (int c = lane; c < warps * kVChunks; c += 32) t += s.chunk_sum[c / kVChunks][c % kVChunks];
                t = warp_sum_f64(t);
                if (lane < (int)ranks) {
                    const uint32_t at = mapa_shared(smem_u32(&s.sum[meeting & 1][rank]), lane);
                    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(t) : "memory");
                }
            }
            if (ranks > 1)
                cluster_sync();
            else
                __syncthreads();
            ++meeting;
        }
        double* sums = s.sum[(meeting & 1) ^ 1];
        if (rejected >= 0) {
            if (tid == 0) {
                double total = 0.0;
                for (int c = 0; c < (int)ranks; ++c) total += sums[c];
                s.summed = node;
                if (rank == 0 && !(fabs(total) < INFINITY)) record_status(a.status, KZ_ERR_NONFINITE);
                if (!q) {
                    take_out(s, rejected, total);
                } else if (total > 0.0) {
                    s.c += s.t;
                    s.t = total;
                    ++s.rejections;
                } else {
                    s.summed = -1;
                }
            }
            continue;
        }
        // the next token: the slice, then the chunk, then the value in which the running sum passes u * total
        if (!q && s.rejections > 0) {
            // without the tokens taken out.  n subtractions leave up to n^2 2^-53 of the largest of them where
            // there is nothing left, which u = 0 would take for mass: as little is none
            __syncthreads();
            if (tid == 0) {
                const int of = warps * kVChunks;
                const double lim = 2.220446049250313e-16 * s.rejections * s.rejections;
                for (int turn = 0; turn < 2; ++turn)
                    for (int k = 0; k < s.rejections; ++k) {
                        const int c = s.gone[k] / a.chunk;
                        const double p = s.gone_p[k];
                        auto take = [&](double& x) { x = turn == 0 ? x - p : x > lim * p ? x : 0.0; };
                        take(sums[c / of]);
                        if (c / of == (int)rank) take(s.chunk_sum[c % of / kVChunks][c % kVChunks]);
                    }
            }
            __syncthreads();
        }
        double total = 0.0;
        for (int c = 0; c < (int)ranks; ++c) total += sums[c];
        const double want = sample_u * total;
        if (rank == 0 && tid == 0 && !(fabs(want) < INFINITY)) record_status(a.status, KZ_ERR_NONFINITE);
        double before = 0.0;
        int slice = -1, last = (int)ranks - 1;
        for (int c = 0; c < (int)ranks; ++c) {
            if (sums[c] > 0.0) last = c;
            if (slice < 0 && before + sums[c] > want) slice = c;
            if (slice < 0) before += sums[c];
        }
        const bool past = slice < 0;                        // u * total at or past the total's rounding: the last value
        if (past) slice = last;
        if (slice == (int)rank && warp == 0) {
            // running sums over the slice's chunks, two a lane
            static_assert(kVWarps * kVChunks <= 64, "two chunks a lane");
            const int n = warps * kVChunks;
            const double t0 = s.chunk_sum[lane / kVChunks][lane % kVChunks];
            const double t1 = n > 32 ? s.chunk_sum[lane / kVChunks + 32 / kVChunks][lane % kVChunks] : 0.0;
            double run0 = t0, run1 = t1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v0 = __shfl_up_sync(0xffffffffu, run0, o), v1 = __shfl_up_sync(0xffffffffu, run1, o);
                if (lane >= o) {
                    run0 += v0;
                    run1 += v1;
                }
            }
            const double first = before + __shfl_sync(0xffffffffu, run0, 31);
            const unsigned hit0 = past ? 0u : __ballot_sync(0xffffffffu, before + run0 > want);
            const unsigned hit1 = past ? 0u : __ballot_sync(0xffffffffu, n > 32 && first + run1 > want);
            const unsigned some0 = __ballot_sync(0xffffffffu, t0 > 0.0), some1 = __ballot_sync(0xffffffffu, t1 > 0.0);
            const bool over = !(hit0 | hit1);               // rounding: the last chunk that has anything
            const int part = hit0 ? __ffs(hit0) - 1 : hit1 ? 31 + __ffs(hit1) : some1 ? 63 - __clz(some1) : some0 ? 31 - __clz(some0) : n - 1;
            const double up0 = __shfl_sync(0xffffffffu, run0, (part - 1) & 31), up1 = __shfl_sync(0xffffffffu, run1, (part - 1) & 31);
            double base = part == 0 ? before : part <= 32 ? before + up0 : first + up1;
            const int plo = (int)min((int64_t)a.vocab, (int64_t)slice0 + (int64_t)part * a.chunk);
            const int phi = (int)min((int64_t)a.vocab, (int64_t)plo + a.chunk);
            int token = -1, top = -1;                       // the answer; the last value above 0
            for (int i0 = plo; i0 < phi && token < 0; i0 += 128) {
                const int i = i0 + 4 * lane;
                const float4 pv = four(p, min(i, phi), phi, a.wide);
                const float4 qv = c_now != 0.0 ? four(q, min(i, phi), phi, a.wide) : make_float4(0.f, 0.f, 0.f, 0.f);
                double r[4], run = 0.0;
                values(pv, qv, r);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!q && is_gone(s, i + e)) r[e] = 0.0;
                    run += r[e];
                }
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += v;
                }
                double at = __shfl_up_sync(0xffffffffu, run, 1);
                at = base + (lane > 0 ? at : 0.0);
                int hit = -1, some = -1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    at += r[e];
                    if (i + e < phi) {
                        if (hit < 0 && !over && at > want) hit = i + e;
                        if (r[e] > 0.0) some = i + e;
                    }
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), somes = __ballot_sync(0xffffffffu, some >= 0);
                if (hits) token = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
                if (somes) top = __shfl_sync(0xffffffffu, some, 31 - __clz(somes));
                base += __shfl_sync(0xffffffffu, run, 31);
            }
            if (lane == 0) a.next[b] = token >= 0 ? token : top >= 0 ? top : a.vocab - 1;
        }
        break;
    }
    if (rank == 0 && tid == 0) a.count[b] = accepted;
    // a CTA's shared memory takes the others' sums: none leaves before all have written
    if (ranks > 1) cluster_sync();
}

}  // namespace
}  // namespace kz

using namespace kz;

extern "C" int kz_verify_tree_f32(const int64_t* tokens, const int32_t* parents, int64_t parents_batch_stride,
                                  const float* target, const float* draft, const float* accept_u,
                                  const float* sample_u, int64_t batch, int64_t nodes, int64_t vocab, int32_t* path,
                                  int32_t* count, int64_t* next, kz_stream_t stream) {
    KZ_REQUIRE(batch >= 0 && batch < (1 << 24), "kz_verify_tree_f32: batch out of range");
    KZ_REQUIRE(nodes >= 1 && nodes <= kVMaxNodes, "kz_verify_tree_f32: nodes must be 1 to 1024");
    KZ_REQUIRE(vocab >= 1 && vocab < (1 << 24), "kz_verify_tree_f32: vocab must be 1 to 2^24 - 1");
    if (batch == 0) return KZ_OK;
    KZ_REQUIRE(tokens && parents && target && accept_u && sample_u && path && count && next,
               "kz_verify_tree_f32: NULL operand");
    KZ_REQUIRE(parents_batch_stride == 0 || parents_batch_stride >= nodes,
               "kz_verify_tree_f32: parents_batch_stride is shorter than nodes");
    int st = check_device();
    if (st) return st;
    VerifyArgs a;
    a.tokens = tokens;
    a.parents = parents;
    a.parents_bs = parents_batch_stride;
    a.target = target;
    a.draft = draft;
    a.accept_u = accept_u;
    a.sample_u = sample_u;
    a.path = path;
    a.count = count;
    a.next = next;
    a.nodes = (int)nodes;
    a.vocab = (int)vocab;
    a.status = device_status_ptr();
    // a cluster for each sequence: the CTAs it takes to have 128 values a warp's chunk, 8 at most; a small
    // vocabulary is one CTA of four warps (65 tokens: 10.4 us, with eight warps 10.6)
    const int threads = vocab <= 4 * kVChunks * 128 ? 128 : kVThreads, warps = threads / 32;
    int ranks = 1;
    while (ranks < kVMaxCluster && vocab > (int64_t)ranks * warps * kVChunks * 128) ranks *= 2;
    const int64_t chunks = (int64_t)ranks * warps * kVChunks;
    a.chunk = (int)((vocab + chunks * 128 - 1) / (chunks * 128)) * 128;
    a.wide = vocab % 4 == 0 && ((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) & 15u) == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * ranks));
    cfg.blockDim = dim3(threads);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    KZ_CHECK_CUDA(cudaLaunchKernelEx(&cfg, verify_tree_kernel, a));
    return KZ_OK;
}
