// Attention over the paged int8 K/V cache: single tokens, chunks of a prompt,
// trees of drafted tokens.
//
//   s_l = (q . c_l) * ks_l / sqrt(d)      c_l, ks_l: key l's codes and scale
//   o   = sum_l w_l * (vs_l * cv_l),  w = softmax(s) over the visible keys
//
// The new tokens' own K/V are in the cache already (positions length ..
// length + count - 1).  New token t sees every token before the new ones, and
// of the new ones its ancestors and itself in the tree (parents) or, without
// a tree, every one up to itself.  Rows past a sequence's count are 0.
#include <math.h>

#include <algorithm>

#include "kz_cache.cuh"

namespace kz {
namespace {

constexpr int kCaThreads = 128;

struct CacheAttArgs {
    CacheView c;
    SeqView s;
    const float* q;
    int64_t q_bs, q_rs;
    const int32_t* counts;
    const int32_t* parents;
    int64_t parents_bs;
    float* out;
    int batch, tokens, heads, group;
    float scale;
    int* status;
};

// A warp a (sequence, new token, head): one pass over the keys with the
// running maximum and sum.
template <int D>
__global__ void __launch_bounds__(kCaThreads) cache_attention_kernel(CacheAttArgs a) {
    constexpr int E = D / 32;
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * (kCaThreads / 32) + (threadIdx.x >> 5);
    if (item >= (int64_t)a.batch * a.tokens * a.heads) return;
    const int h = (int)(item % a.heads);
    const int64_t bt = item / a.heads;
    const int t = (int)(bt % a.tokens);
    const int64_t b = bt / a.tokens;
    const int count = a.counts ? min(a.counts[b], a.tokens) : a.tokens;
    const int64_t len = min((int64_t)max(0, a.s.lengths[b]), (int64_t)a.s.cols * a.c.page);
    const int32_t* parents = a.parents ? a.parents + b * a.parents_bs : nullptr;
    const int kvh = h / a.group;
    float q[E], o[E], m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = a.q[b * a.q_bs + t * a.q_rs + (int64_t)h * D + lane * E + e] * a.scale;
        o[e] = 0.0f;
    }
    int anc = t;   // the next visible node at or below the current one, walking up from t
    if (t < count) {
        for (int64_t l = len + t; l >= 0; --l) {
            if (parents && l >= len) {
                if (l - len != anc) continue;
                const int up = parents[anc];
                anc = up < anc ? up : -1;
            }
            const int page = page_of(a.c, a.s, b, l);
            if (page < 0) {
                if (lane == 0) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
                continue;
            }
            const int64_t row = ((int64_t)page * a.c.heads + kvh) * a.c.page + (l & (a.c.page - 1));
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) s += q[e] * (float)a.c.codes[0][row * D + lane * E + e];
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            s *= a.c.scale[0][row];
            const float top = fmaxf(m, s);
            const float keep = expf(m - top), w = expf(s - top), vs = w * a.c.scale[1][row];
            m = top;
            sum = sum * keep + w;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = o[e] * keep + vs * (float)a.c.codes[1][row * D + lane * E + e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        a.out[bt * a.heads * D + (int64_t)h * D + lane * E + e] = sum > 0.0f ? o[e] / sum : 0.0f;
}

}  // namespace
}  // namespace kz

using namespace kz;

extern "C" int kz_cache_attention_f32(const kz_cache* cache, const float* q, int64_t batch, int64_t tokens,
                                      int64_t heads, int64_t q_batch_stride, int64_t q_row_stride,
                                      const int32_t* table, int64_t table_cols, const int32_t* lengths,
                                      const int32_t* counts, const int32_t* parents, int64_t parents_batch_stride,
                                      float scale, float* out, kz_stream_t stream) {
    CacheAttArgs a;
    int st = cache_view(cache, "kz_cache_attention_f32", &a.c);
    if (!st) st = seq_view(table, table_cols, lengths, batch, "kz_cache_attention_f32", &a.s);
    if (st) return st;
    KZ_REQUIRE(heads > 0 && heads % cache->kv_heads == 0,
               "kz_cache_attention_f32: heads must be a multiple of kv_heads");
    KZ_REQUIRE(tokens >= 0 && tokens < (1 << 24) && batch * tokens * heads < (int64_t)INT32_MAX,
               "kz_cache_attention_f32: size out of range");
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
    st = check_device();
    if (st) return st;
    a.q = q;
    a.q_bs = q_batch_stride;
    a.q_rs = q_row_stride;
    a.counts = counts;
    a.parents = parents;
    a.parents_bs = parents_batch_stride;
    a.out = out;
    a.batch = (int)batch;
    a.tokens = (int)tokens;
    a.heads = (int)heads;
    a.group = (int)(heads / cache->kv_heads);
    a.scale = scale;
    a.status = device_status_ptr();
    const int64_t warps = batch * tokens * heads;
    const dim3 grid((unsigned)((warps + kCaThreads / 32 - 1) / (kCaThreads / 32)));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    auto kernel = cache->head_dim == 32   ? cache_attention_kernel<32>
                  : cache->head_dim == 64 ? cache_attention_kernel<64>
                                          : cache_attention_kernel<128>;
    KZ_CHECK_CUDA(launch_pdl(kernel, grid, dim3(kCaThreads), 0, s, a));
    return KZ_OK;
}
