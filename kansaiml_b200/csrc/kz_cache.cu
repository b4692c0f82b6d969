// The paged int8 K/V cache: writing new tokens, reading tokens back, moving
// the accepted path of a drafted tree to the front.
//
// A token's head (d values) is one row with its own scale, quantized by the
// framework's rule (kz_quant_math.cuh): scale = max|x| / 127 in double (1 for
// a row of zeros), code = rint(x / scale) half to even.  What is kept is the
// code and fl32(scale); a cached value stands for fl32(code * fl32(scale)).
//
// All three kernels move each byte once and are bound by HBM (small calls by
// the launch).  A page keeps each head's slots together ([page][head][slot][d]),
// so attention and the read-back stream whole pages; a written row is d
// contiguous bytes.
#include <algorithm>

#include "kz_cache.cuh"
#include "kz_quant_math.cuh"

namespace kz {
namespace {

constexpr int kCacheThreads = 256;

struct WriteArgs {
    CacheView c;
    SeqView s;
    const float* x[2];                 // K, V
    int64_t bs[2], rs[2];              // batch and row strides (floats)
    float* values[2];                  // what the codes stand for, [batch, tokens, heads * d], or NULL
    const int32_t* counts;
    uint32_t tokens, items;            // items = batch * tokens * groups of heads
    FastDiv by_groups, by_tokens;
    int* status;
};

// Four codes (a packed word) as floats times a scale, one rounding each: the
// byte, offset by 128, in the mantissa of 2^23, less 2^23 + 128, is the code.
__device__ __forceinline__ float4 codes_times(uint32_t w, float s) {
    w ^= 0x80808080u;
    float4 v;
    v.x = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440)) - 8388736.0f, s);
    v.y = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441)) - 8388736.0f, s);
    v.z = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7442)) - 8388736.0f, s);
    v.w = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7443)) - 8388736.0f, s);
    return v;
}

// A warp takes a token's next kU * G heads: G groups of D / 4 lanes (16 bytes a
// lane) hold a row each, K and V of kU such row sets are in flight.  What
// depends on the token alone (its page, its slot) is found once a warp.  The
// rows' scales need two double divisions each: they are handed to one lane a
// row and back by shuffles, so a warp divides once for all its rows.  Bound by
// HBM: 16 prompts of up to 2000 tokens, 8 heads of 128, values returned (509
// MB), 88 us = 5.8 TB/s, 0.89 of a plain copy; a row at a time, every row
// finding its own place and dividing for itself, took 208 us.  Without values (247
// MB) 57 us = 4.3 TB/s, 0.66: there the quantizing, which those writes hid, shows.
// One token of 32 sequences, 4 heads of 64: 3.0 us, the launch.
template <int D, int kU>
__global__ void __launch_bounds__(kCacheThreads, 4) cache_write_kernel(WriteArgs a) {
    constexpr int L = D / 4, G = 32 / L, N = 2 * kU * G;   // lanes a row, groups a warp, rows a warp
    static_assert(N <= 32, "a lane for each row's scale");
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, sub = lane / L, col = 4 * (lane % L);
    const uint32_t item = blockIdx.x * (kCacheThreads / 32) + __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    if (item >= a.items) return;
    const uint32_t bt = div_by(item, a.by_groups), h0 = (item - bt * a.by_groups.d) * (kU * G) + sub;   // u adds u * G
    const uint32_t b = div_by(bt, a.by_tokens), t = bt - b * a.by_tokens.d;
    const int64_t out_at = ((int64_t)bt * a.c.heads + h0) * D + col;
    if (a.counts && (int)t >= a.counts[b]) {               // padding: its values are 0
#pragma unroll
        for (int i = 0; i < 2 * kU; ++i)
            if (h0 + (i >> 1) * G < (uint32_t)a.c.heads && a.values[i & 1])
                __stcs(reinterpret_cast<float4*>(a.values[i & 1] + out_at + (i >> 1) * G * D), make_float4(0.f, 0.f, 0.f, 0.f));
        return;
    }
    float4 x[2 * kU];
    uint32_t bits[2 * kU];
#pragma unroll
    for (int i = 0; i < 2 * kU; ++i) {
        const int kv = i & 1;
        const uint32_t h = h0 + (i >> 1) * G;
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < (uint32_t)a.c.heads)
            x[i] = __ldcs(reinterpret_cast<const float4*>(a.x[kv] + b * a.bs[kv] + t * a.rs[kv] + h * D + col));
    }
    const int64_t pos = (int64_t)a.s.lengths[b] + t;
    const int page = page_of(a.c, a.s, b, pos);
    if (page < 0 && lane == 0) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
    const int64_t row_at = ((int64_t)page * a.c.heads + h0) * a.c.page + (pos & (a.c.page - 1));
#pragma unroll
    for (int i = 0; i < 2 * kU; ++i) {
        uint32_t m = max(max(abs_bits(x[i].x), abs_bits(x[i].y)), max(abs_bits(x[i].z), abs_bits(x[i].w)));
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        bits[i] = m;
    }
    // lane i * G + g: the scale of row set i of group g
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 2 * kU; ++i) {
        const uint32_t m = G == 1 ? bits[i] : __shfl_sync(0xffffffffu, bits[i], (lane % G) * L);
        if (lane / G == i) mine = m;
    }
    const ScaleInfo si = scale_from_absmax_bits(mine);
    const float s32 = si.finite ? __double2float_rn(si.scale) : __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int i = 0; i < 2 * kU; ++i) {
        const int u = i >> 1, kv = i & 1;
        const float s = __shfl_sync(0xffffffffu, s32, i * G + sub);
        const float rcp = __shfl_sync(0xffffffffu, si.rcp, i * G + sub);
        if (h0 + u * G >= (uint32_t)a.c.heads) continue;
        uint32_t w = 0;
        if (bits[i] - 1 < kInfBits - 1) {            // neither zeros nor NaN/Inf, whose codes are 0
            const bool fast = bits[i] >= __float_as_uint(7.8886090522101181e-31f);   // as scale_from_absmax_bits has it
            float near;
            w = pack4_fast(x[i], rcp, near);
            if (!fast || near > kTieGuardFma)
                w = pack4_repair(x[i], w, scale_from_absmax_bits(bits[i]).scale, rcp, fast);
        }
        if (page >= 0) {
            const int64_t row = row_at + (int64_t)u * G * a.c.page;
            *reinterpret_cast<uint32_t*>(a.c.codes[kv] + row * D + col) = w;
            if (col == 0) {
                a.c.scale[kv][row] = s;
                if (bits[i] >= kInfBits) record_status(a.status, KZ_ERR_NONFINITE);
            }
        }
        if (a.values[kv]) __stcs(reinterpret_cast<float4*>(a.values[kv] + out_at + u * G * D), codes_times(w, s));
    }
}

struct ReadArgs {
    CacheView c;
    SeqView s;
    float* out[2];                     // [batch, most, heads * d]
    uint32_t most, chunks, items;      // items = batch * chunks (pages up to `most`) * heads
    FastDiv by_heads, by_chunks;
    int* status;
};

// A warp a (sequence, page, head): streams the page's K and V slots of that
// head (contiguous) and writes rows of d floats; rows past the sequence's
// length are written as zeros.  Four code words of K and four of V in flight.
// Bound by HBM, four fifths of it the fp32 rows written (past the caches, which
// they would only empty): 8 sequences of 8000 to 16000 tokens, 8 heads of 128
// (1.25 GB), 220 us = 5.7 TB/s, 0.87 of a plain copy.
template <int D>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(ReadArgs a) {
    constexpr int L = D / 4, G = 32 / L;
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, sub = lane / L, col = 4 * (lane % L);
    const uint32_t item = blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5);
    if (item >= a.items) return;
    const uint32_t bc = div_by(item, a.by_heads), h = item - bc * a.by_heads.d;
    const uint32_t b = div_by(bc, a.by_chunks), chunk = bc - b * a.by_chunks.d;
    const int64_t first = (int64_t)chunk * a.c.page;
    const int rows = (int)min((int64_t)a.c.page, (int64_t)a.most - first);          // output rows of this page
    const int length = a.s.lengths[b];
    int held = (int)min((int64_t)rows, max((int64_t)0, (int64_t)length - first));
    if (length < 0 && lane == 0) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
    int64_t base = 0;
    if (held > 0) {
        const int page = page_of(a.c, a.s, b, first);
        if (page < 0) {
            if (lane == 0) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
            held = 0;
        }
        base = ((int64_t)page * a.c.heads + h) * a.c.page;
    }
    const int64_t width = (int64_t)a.c.heads * D;
    const int64_t out_at = ((int64_t)b * a.most + first) * width + h * D + col;
    for (int r0 = 0; r0 < rows; r0 += 4 * G) {
        uint32_t w[2][4];
        float s[2][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = r0 + u * G + sub;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const bool there = r < held;
                w[kv][u] = there ? __ldcs(reinterpret_cast<const uint32_t*>(a.c.codes[kv] + (base + r) * D + col)) : 0u;
                s[kv][u] = there ? __ldg(a.c.scale[kv] + base + r) : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = r0 + u * G + sub;
            if (r < rows) {
#pragma unroll
                for (int kv = 0; kv < 2; ++kv)
                    __stcs(reinterpret_cast<float4*>(a.out[kv] + out_at + r * width), codes_times(w[kv][u], s[kv][u]));
            }
        }
    }
}

struct KeepArgs {
    CacheView c;
    SeqView s;
    const int32_t* path;               // [batch, nodes]
    const int32_t* count;              // [batch]
    int batch, nodes;
    int* status;
};

// A warp a (sequence, head): slot length + path[i] moves to length + i.  A
// path is strictly increasing (a node comes after its parent), so path[i] >= i
// and a row's new slot is never the old slot of a later row: passes of whole
// rows, every load of a pass before its stores, move in place without a copy.
// A path that is not strictly increasing within [0, nodes) moves nothing.
// Latency bounds it (length, path, table, row, one after another): 32 trees of
// 6 nodes, 4 heads of 64, 2.4 us; 128 of 64 nodes, 8 heads of 128, 5.4 us.
template <int D>
__global__ void __launch_bounds__(kCacheThreads) cache_keep_kernel(KeepArgs a) {
    constexpr int L = D / 16, G = 32 / L;    // 16 codes a lane
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, sub = lane / L, col = 16 * (lane % L);
    const int64_t item = (int64_t)blockIdx.x * (kCacheThreads / 32) + (threadIdx.x >> 5);
    if (item >= (int64_t)a.batch * a.c.heads) return;
    const int b = (int)(item / a.c.heads), h = (int)(item % a.c.heads);
    const int32_t* path = a.path + (int64_t)b * a.nodes;
    const int n = a.count[b];
    const int64_t len = a.s.lengths[b];
    bool good = n >= 0 && n <= a.nodes;
    if (good)
        for (int i = lane; i < n; i += 32)
            good = good && path[i] >= (i > 0 ? path[i - 1] + 1 : 0) && path[i] < a.nodes &&
                   page_of(a.c, a.s, b, len + i) >= 0 && page_of(a.c, a.s, b, len + path[i]) >= 0;
    if (!__all_sync(0xffffffffu, good)) {
        if (lane == 0) record_status(a.status, KZ_ERR_INVALID_ARGUMENT);
        return;
    }
    for (int i0 = 0; i0 < n; i0 += G) {
        const int i = i0 + sub;
        const bool moves = i < n && path[i] != i;
        int64_t from = 0, to = 0;
        uint4 w[2];
        float s[2];
        if (moves) {
            const int64_t p = len + path[i], q = len + i;
            from = ((int64_t)page_of(a.c, a.s, b, p) * a.c.heads + h) * a.c.page + (p & (a.c.page - 1));
            to = ((int64_t)page_of(a.c, a.s, b, q) * a.c.heads + h) * a.c.page + (q & (a.c.page - 1));
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                w[kv] = *reinterpret_cast<const uint4*>(a.c.codes[kv] + from * D + col);
                s[kv] = a.c.scale[kv][from];
            }
        }
        __syncwarp();
        if (moves) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                *reinterpret_cast<uint4*>(a.c.codes[kv] + to * D + col) = w[kv];
                if (col == 0) a.c.scale[kv][to] = s[kv];
            }
        }
        __syncwarp();
    }
}

// Row sets a warp holds: as many as the heads fill, four at most.  With 1, 2
// and 4 sets, heads of 128, 16 x 2000 tokens: 1 head 14.6, 16.1, 20.5 us; 2
// heads 29.0, 24.2, 27.2 us; 8 heads 111, 88.9, 87.6 us (without values 66.3 with 2
// and 57.2 with 4).  Heads of 64 and 32, whose four sets spill 44 bytes a thread,
// with 2 and 4: 8 of 64 45.2 and 46.9 us (without values 33.9, 33.1), 16 of 64 88.9,
// 91.6 (65.7, 62.4), 16 of 32 45.8, 50.0 (33.8, 35.2).  32 single tokens, 8 heads of
// any width, are the other way round: 3.0 us with 2 sets, 4.3 with 4.
template <int D>
int launch_write(WriteArgs a, int64_t batch, cudaStream_t s) {
    constexpr int G = 128 / D;
    const int sets = a.c.heads <= G ? 1 : a.c.heads <= 2 * G ? 2 : 4;
    const uint32_t groups = (uint32_t)((a.c.heads + sets * G - 1) / (sets * G));
    a.items = (uint32_t)(batch * a.tokens * groups);
    a.by_groups = fast_div(groups);
    const dim3 grid((a.items + kCacheThreads / 32 - 1) / (kCacheThreads / 32));
    auto kernel = sets == 1 ? cache_write_kernel<D, 1> : sets == 2 ? cache_write_kernel<D, 2> : cache_write_kernel<D, 4>;
    KZ_CHECK_CUDA(launch_pdl(kernel, grid, dim3(kCacheThreads), 0, s, a));
    return KZ_OK;
}

}  // namespace

int cache_view(const kz_cache* c, const char* who, CacheView* v) {
    KZ_REQUIRE(c, std::string(who) + ": cache is NULL");
    KZ_REQUIRE(c->head_dim == 32 || c->head_dim == 64 || c->head_dim == 128, std::string(who) + ": head_dim must be 32, 64 or 128");
    KZ_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
               std::string(who) + ": page_size must be 16, 32, 64 or 128");
    KZ_REQUIRE(c->pages >= 0 && c->kv_heads > 0 && c->kv_heads < (1 << 16) &&
                   c->pages * c->kv_heads < (int64_t)INT32_MAX / c->page_size,
               std::string(who) + ": cache size out of range (pages * kv_heads * page_size must be below 2^31)");
    KZ_REQUIRE(c->pages == 0 || (c->k_codes && c->v_codes && c->k_scale && c->v_scale), std::string(who) + ": NULL cache buffer");
    const uintptr_t bits = reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes) |
                           reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale);
    KZ_REQUIRE((bits & 15u) == 0, std::string(who) + ": cache buffers must be 16-byte aligned");
    v->codes[0] = c->k_codes;
    v->codes[1] = c->v_codes;
    v->scale[0] = c->k_scale;
    v->scale[1] = c->v_scale;
    v->pages = (int)c->pages;
    v->heads = (int)c->kv_heads;
    v->page = (int)c->page_size;
    v->shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    return KZ_OK;
}

int seq_view(const int32_t* table, int64_t cols, const int32_t* lengths, int64_t batch, const char* who, SeqView* v) {
    KZ_REQUIRE(batch >= 0 && batch < (1 << 24) && cols >= 0 && cols < (1 << 24), std::string(who) + ": batch or table size out of range");
    KZ_REQUIRE(batch == 0 || ((table || cols == 0) && lengths), std::string(who) + ": table or lengths is NULL");
    v->table = table;
    v->lengths = lengths;
    v->cols = (int)cols;
    return KZ_OK;
}

}  // namespace kz

using namespace kz;

extern "C" int kz_cache_write_f32(const kz_cache* cache, const float* k, const float* v, int64_t batch, int64_t tokens,
                                  int64_t k_batch_stride, int64_t k_row_stride, int64_t v_batch_stride,
                                  int64_t v_row_stride, const int32_t* table, int64_t table_cols,
                                  const int32_t* lengths, const int32_t* counts, float* k_values, float* v_values,
                                  kz_stream_t stream) {
    WriteArgs a;
    int st = cache_view(cache, "kz_cache_write_f32", &a.c);
    if (!st) st = seq_view(table, table_cols, lengths, batch, "kz_cache_write_f32", &a.s);
    if (st) return st;
    const int64_t width = cache->kv_heads * cache->head_dim;
    KZ_REQUIRE(tokens >= 0 && tokens < (1 << 24), "kz_cache_write_f32: tokens out of range");
    KZ_REQUIRE(batch * tokens < (int64_t)INT32_MAX / cache->kv_heads, "kz_cache_write_f32: batch * tokens * kv_heads out of range");
    if (batch * tokens == 0) return KZ_OK;
    KZ_REQUIRE(k && v, "kz_cache_write_f32: k or v is NULL");
    const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                           reinterpret_cast<uintptr_t>(k_values) | reinterpret_cast<uintptr_t>(v_values);
    KZ_REQUIRE((bits & 15u) == 0 && ((k_batch_stride | k_row_stride | v_batch_stride | v_row_stride) & 3) == 0,
               "kz_cache_write_f32: k, v and the values must be 16-byte aligned, strides multiples of 4 floats");
    KZ_REQUIRE(tokens == 1 || (k_row_stride >= width && v_row_stride >= width),
               "kz_cache_write_f32: a row stride is shorter than kv_heads * head_dim");
    KZ_REQUIRE(k_batch_stride >= 0 && v_batch_stride >= 0, "kz_cache_write_f32: negative batch stride");
    st = check_device();
    if (st) return st;
    a.x[0] = k;
    a.x[1] = v;
    a.bs[0] = k_batch_stride;
    a.bs[1] = v_batch_stride;
    a.rs[0] = k_row_stride;
    a.rs[1] = v_row_stride;
    a.values[0] = k_values;
    a.values[1] = v_values;
    a.counts = counts;
    a.tokens = (uint32_t)tokens;
    a.by_tokens = fast_div((uint32_t)tokens);
    a.status = device_status_ptr();
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return cache->head_dim == 32   ? launch_write<32>(a, batch, s)
           : cache->head_dim == 64 ? launch_write<64>(a, batch, s)
                                   : launch_write<128>(a, batch, s);
}

extern "C" int kz_cache_read_f32(const kz_cache* cache, const int32_t* table, int64_t table_cols,
                                 const int32_t* lengths, int64_t batch, int64_t most, float* k_out, float* v_out,
                                 kz_stream_t stream) {
    ReadArgs a;
    int st = cache_view(cache, "kz_cache_read_f32", &a.c);
    if (!st) st = seq_view(table, table_cols, lengths, batch, "kz_cache_read_f32", &a.s);
    if (st) return st;
    KZ_REQUIRE(most >= 0 && most < (int64_t)INT32_MAX, "kz_cache_read_f32: most out of range");
    if (batch * most == 0) return KZ_OK;
    const int64_t chunks = (most + cache->page_size - 1) / cache->page_size;
    KZ_REQUIRE(batch * chunks < (int64_t)INT32_MAX / cache->kv_heads, "kz_cache_read_f32: batch * most * kv_heads out of range");
    KZ_REQUIRE(k_out && v_out, "kz_cache_read_f32: k_out or v_out is NULL");
    KZ_REQUIRE(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u) == 0,
               "kz_cache_read_f32: k_out and v_out must be 16-byte aligned");
    st = check_device();
    if (st) return st;
    a.out[0] = k_out;
    a.out[1] = v_out;
    a.most = (uint32_t)most;
    a.chunks = (uint32_t)chunks;
    a.items = (uint32_t)(batch * chunks * cache->kv_heads);
    a.by_heads = fast_div((uint32_t)cache->kv_heads);
    a.by_chunks = fast_div((uint32_t)chunks);
    a.status = device_status_ptr();
    const dim3 grid((a.items + kCacheThreads / 32 - 1) / (kCacheThreads / 32));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    auto kernel = cache->head_dim == 32 ? cache_read_kernel<32> : cache->head_dim == 64 ? cache_read_kernel<64>
                                                                                       : cache_read_kernel<128>;
    KZ_CHECK_CUDA(launch_pdl(kernel, grid, dim3(kCacheThreads), 0, s, a));
    return KZ_OK;
}

extern "C" int kz_cache_keep(const kz_cache* cache, const int32_t* table, int64_t table_cols, const int32_t* lengths,
                             const int32_t* path, const int32_t* count, int64_t batch, int64_t nodes,
                             kz_stream_t stream) {
    KeepArgs a;
    int st = cache_view(cache, "kz_cache_keep", &a.c);
    if (!st) st = seq_view(table, table_cols, lengths, batch, "kz_cache_keep", &a.s);
    if (st) return st;
    KZ_REQUIRE(nodes >= 0 && nodes < (1 << 24), "kz_cache_keep: nodes out of range");
    KZ_REQUIRE(batch < (int64_t)INT32_MAX / cache->kv_heads, "kz_cache_keep: batch * kv_heads out of range");
    if (batch * nodes == 0) return KZ_OK;
    KZ_REQUIRE(path && count, "kz_cache_keep: path or count is NULL");
    st = check_device();
    if (st) return st;
    a.path = path;
    a.count = count;
    a.batch = (int)batch;
    a.nodes = (int)nodes;
    a.status = device_status_ptr();
    const int64_t warps = batch * cache->kv_heads;
    const dim3 grid((unsigned)((warps + kCacheThreads / 32 - 1) / (kCacheThreads / 32)));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    auto kernel = cache->head_dim == 32 ? cache_keep_kernel<32> : cache->head_dim == 64 ? cache_keep_kernel<64>
                                                                                       : cache_keep_kernel<128>;
    KZ_CHECK_CUDA(launch_pdl(kernel, grid, dim3(kCacheThreads), 0, s, a));
    return KZ_OK;
}
