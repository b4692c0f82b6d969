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
// Everything is computed in double from the fp32 rows, so that the decisions
// do not depend on how the work is split.
//
// Each sequence is walked by one cluster: every CTA takes a slice of the
// vocabulary and repeats the walk itself (the accept tests need single values
// only, gathered up front), so that the cluster meets once a rejection and
// once at the end, to exchange the slices' sums through distributed shared
// memory.  A rejection reads two rows (one without a draft), the last token
// the same rows once more; nothing else of the probabilities is touched.
#include <math.h>

#include <algorithm>

#include "kz_common.cuh"

namespace kz {
namespace {

constexpr int kVThreads = 512, kVWarps = kVThreads / 32;
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
    int nodes, vocab, per;     // per: values a CTA's slice holds (a multiple of 128 * warps)
    int* status;
};

struct VerifyShared {
    double sum[2][kVMaxCluster];       // the slices' sums, a buffer for each of two successive meetings
    double warp_sum[kVWarps];
    double scale[kVMaxNodes];          // 1 / sum of each rejection at the current node
    float p_at[kVMaxNodes], q_at[kVMaxNodes], u[kVMaxNodes];
    int parent[kVMaxNodes], token[kVMaxNodes];
    int gone[kVMaxNodes];              // no draft: the tokens rejected at the current node
    int rejections, node, child, found;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// r at token i, from the target's and the draft's value there
__device__ __forceinline__ double rest_at(const VerifyShared& s, bool has_draft, int i, float p, float q) {
    double r = p;
    for (int k = 0; k < s.rejections; ++k) {
        if (has_draft)
            r = fmax(r - (double)q, 0.0) * s.scale[k];
        else
            r = s.gone[k] == i ? 0.0 : r * s.scale[k];
    }
    return r;
}

__global__ void __launch_bounds__(kVThreads) verify_tree_kernel(VerifyArgs a) {
    __shared__ VerifyShared s;
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
    const int64_t b = blockIdx.x / ranks;
    const float* target = a.target + b * a.nodes * (int64_t)a.vocab;
    const float* draft = a.draft ? a.draft + b * a.nodes * (int64_t)a.vocab : nullptr;
    for (int j = tid; j < a.nodes; j += kVThreads) {
        int parent = a.parents[b * a.parents_bs + j];
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
        s.child = 1;
        s.found = -1;
    }
    int accepted = 1, meeting = 0;
    const int lo = (int)rank * a.per, hi = min(a.vocab, lo + a.per);
    const int span = a.per / kVWarps;                       // a warp's part of the slice
    const int wlo = min(hi, lo + warp * span), whi = min(hi, wlo + span);
    for (;;) {
        __syncthreads();
        if (tid == 0) {
            // walk to the next rejection (s.found: the rejected child) or past the last node
            s.found = -1;
            int j = s.child;
            for (; j < a.nodes; ++j) {
                if (s.parent[j] != s.node) continue;
                const double r = rest_at(s, draft != nullptr, s.token[j], s.p_at[j], s.q_at[j]);
                if ((double)s.u[j] * (double)s.q_at[j] < r) {
                    s.node = j;
                    s.rejections = 0;
                    if (rank == 0) a.path[b * a.nodes + accepted] = j;
                    ++accepted;
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
        const int x = rejected >= 0 ? s.token[rejected] : -1;
        // the sum of this slice: of (r - q)+ after a rejection, of r at the end
        double sum = 0.0;
        for (int i = wlo + lane; i < whi; i += 32) {
            const float qi = q ? q[i] : 0.0f;
            double r = rest_at(s, q != nullptr, i, p[i], qi);
            if (rejected >= 0) r = q ? fmax(r - (double)qi, 0.0) : i == x ? 0.0 : r;
            sum += r;
        }
        sum = warp_sum_f64(sum);
        if (lane == 0) s.warp_sum[warp] = sum;
        __syncthreads();
        if (tid < (int)ranks) {
            double t = 0.0;
            for (int w = 0; w < kVWarps; ++w) t += s.warp_sum[w];
            const uint32_t at = mapa_shared(smem_u32(&s.sum[meeting & 1][rank]), tid);
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(t) : "memory");
        }
        cluster_sync();
        const double* sums = s.sum[meeting & 1];
        ++meeting;
        double total = 0.0;
        for (int c = 0; c < (int)ranks; ++c) total += sums[c];
        if (rejected >= 0) {
            if (tid == 0 && total > 0.0) {
                s.scale[s.rejections] = 1.0 / total;
                s.gone[s.rejections] = x;
                ++s.rejections;
            }
            continue;
        }
        // the next token: the slice, then the warp's part, then the value in which the running sum passes u * total
        const double want = (double)a.sample_u[b] * total;
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
            int part = -1, end = kVWarps - 1;
            double base = before;
            for (int w = 0; w < kVWarps; ++w) {
                if (s.warp_sum[w] > 0.0) end = w;
                if (!past && part < 0 && base + s.warp_sum[w] > want) part = w;
                if (!past && part < 0) base += s.warp_sum[w];
            }
            const bool over = part < 0;
            if (over) part = end;
            const int plo = min(hi, lo + part * span), phi = min(hi, plo + span);
            int token = -1, top = -1;                       // the answer; the last value above 0
            for (int i0 = plo; i0 < phi && token < 0; i0 += 32) {
                const int i = i0 + lane;
                const double r = i < phi ? rest_at(s, q != nullptr, i, p[i], q ? q[i] : 0.0f) : 0.0;
                double run = r;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += v;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, !over && i < phi && base + run > want);
                const unsigned some = __ballot_sync(0xffffffffu, r > 0.0);
                if (hit) token = i0 + __ffs(hit) - 1;
                if (some) top = i0 + 31 - __clz(some);
                base += __shfl_sync(0xffffffffu, run, 31);
            }
            if (lane == 0) a.next[b] = token >= 0 ? token : top >= 0 ? top : a.vocab - 1;
        }
        break;
    }
    if (rank == 0 && tid == 0) a.count[b] = accepted;
    // a CTA's shared memory takes the others' sums: none leaves before all have written
    cluster_sync();
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
    // a cluster for each sequence: 8 CTAs once a slice has 4 values a thread, fewer for small vocabularies
    int ranks = 1;
    while (ranks < kVMaxCluster && vocab > (int64_t)ranks * kVThreads * 4) ranks *= 2;
    const int unit = 32 * kVWarps;
    a.per = (int)((vocab + (int64_t)ranks * unit - 1) / ((int64_t)ranks * unit)) * unit;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * ranks));
    cfg.blockDim = dim3(kVThreads);
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
