// The rounding rule of the framework's int8 codes, as device functions: the
// scale of an absmax and the codes of one, four or sixteen values.
//
// Rounding contract (bit-exact with the reference): every fp32 element is
// widened to double, scale = (double)max|x| / 127.0 (1.0 if max|x| == 0),
// q = clamp(rint((double)x / scale), -127, 127) with rint rounding half to
// even on the correctly rounded double quotient.
//
// Fast path.  The exact double division per element is replaced by an fp32
// estimate t = fl32(x * r), r = fl32(fl64(1 / scale)).  With |x / scale| <= 127:
//   |r - 1/scale| <= (2^-53 + 2^-24 + 2^-77) / scale
//   |t - x*r|     <= 2^-24 |x*r|   (+2^-149 if t is subnormal)
// so |t - x/scale| < 127 * 2^-22.9 < 2^-16, and the double quotient differs
// from x/scale by at most 128 * 2^-53.  Hence |t - fl64(x/scale)| < 2^-15.
// Whenever t lies at least 2^-15 away from every half-integer
// (|t - rint(t)| <= 1/2 - 2^-15), fl64(x/scale) lies in the same open interval
// (k - 1/2, k + 1/2) and rounds to the same k = rint(t).  The remaining
// elements (about 1 in 2000 for smooth data) take the exact double division.
// t - rint(t) is computed exactly (Sterbenz).  When 1/scale does not fit fp32
// (max|x| < 2^-100) every element takes the exact path.
//
// The fast path rounds with one fp32 add: y = t + 1.5 * 2^23 lies in
// [2^23, 2^24) where floats are the integers, so the add itself rounds t half
// to even, y - 1.5 * 2^23 = rint(t) exactly, and y's bit pattern is
// 0x4B400000 + rint(t), whose low byte is the two's-complement int8 code.  No
// clamp is needed: |t| <= 127 * (1 + 2^-23) * (1 + 2^-24) < 127.5 - 2^-12, so
// rint(t) is in [-127, 127] and never near the 127.5 tie.
//
// The vector form (pack4) folds the multiply into fused multiply-adds:
// y = fl32(x*r + 1.5 * 2^23) gives k = y - 1.5 * 2^23, the integer nearest to
// the exact product x*r, and d = fl32(x*r - k) its residual with one rounding
// (|fl32(d) - d| <= 2^-25).  |x*r - x/scale| <= 127 (1 + 2^-52)(2^-24 + 2^-53
// + 2^-77) < 2^-17.01, so |fl64(x/scale) - k| <= |fl32(d)| + 2^-25 + 2^-17.01
// + 2^-46 < |fl32(d)| + 2^-16.9, and |fl32(d)| <= 1/2 - 2^-16 proves
// k = rint(fl64(x/scale)).  Only the elements that fail the bound (about one in
// 16000 for smooth data) take the exact division.
#pragma once

#include "kz_common.cuh"

namespace kz {

constexpr float kTieGuard = 0.5f - 1.0f / 32768.0f;       // scalar form: |t - rint(t)| bound
constexpr float kTieGuardFma = 0.5f - 1.0f / 65536.0f;    // fused-multiply-add form: |d| bound
constexpr uint32_t kInfBits = 0x7F800000u;

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// ------------------------------------------------------- scale + quantize

struct ScaleInfo {
    double scale;   // the reference's double scale
    float rcp;      // fl32(fl64(1 / scale)), fast-path multiplier
    bool fast;      // fast path valid (1/scale representable in fp32)
    bool finite;    // absmax finite
};

__device__ __forceinline__ ScaleInfo scale_from_absmax_bits(uint32_t bits) {
    ScaleInfo si;
    si.finite = bits < kInfBits;
    const float a = __uint_as_float(bits);
    si.scale = a > 0.0f ? (double)a / 127.0 : 1.0;   // quantize.py:68
    si.rcp = __double2float_rn(1.0 / si.scale);
    si.fast = a >= 7.8886090522101181e-31f;           // 2^-100
    return si;
}

__device__ __forceinline__ int8_t quant_exact(float v, double scale) {
    double t = rint((double)v / scale);               // quantize.py:69, IEEE division
    t = fmin(fmax(t, -127.0), 127.0);
    return (int8_t)(int)t;
}

__device__ __forceinline__ int8_t quant_one(float v, const ScaleInfo& si) {
    if (si.fast) {
        const float t = __fmul_rn(v, si.rcp);
        const float tr = rintf(t);
        if (fabsf(t - tr) <= kTieGuard) return (int8_t)(int)fminf(fmaxf(tr, -127.0f), 127.0f);
    }
    return quant_exact(v, si.scale);
}

constexpr float kRoundMagic = 12582912.0f;   // 1.5 * 2^23

// Code of one element by the fused-multiply-add form (see the file header);
// *near is set when the element needs the exact path.
__device__ __forceinline__ uint32_t fma_code(float v, float rcp, bool* near) {
    const float y = __fmaf_rn(v, rcp, kRoundMagic);
    const float d = __fmaf_rn(v, rcp, -__fsub_rn(y, kRoundMagic));
    *near = fabsf(d) > kTieGuardFma;
    return __float_as_uint(y) & 0xFFu;
}

// Exact-path repair of a packed word: only the near-tie bytes are recomputed,
// so a warp with one such element pays for one division.
__device__ __forceinline__ uint32_t pack4_repair(float4 v, uint32_t w, double scale, float rcp, bool fast) {
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        bool near = true;
        if (fast) fma_code(e[j], rcp, &near);
        if (near) w = (w & ~(0xFFu << (8 * j))) | ((uint32_t)(uint8_t)quant_exact(e[j], scale) << (8 * j));
    }
    return w;
}

// Packed fp32 pairs (sm_100 f32x2 arithmetic: each lane rounds exactly like
// the scalar instruction, so results are bit-identical).
__device__ __forceinline__ uint64_t pk2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void upk2(uint64_t r, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Fast-path word of four codes (little-endian) and the largest |residual| of
// the four; residuals above kTieGuardFma mark elements for pack4_repair.
// Per pair: y = fl(x*r + M), -k = M - y (exact), d = fl(x*r - k).
__device__ __forceinline__ uint32_t pack4_fast(const float4& v, float rcp, float& dmax) {
    const uint64_t R = pk2(rcp, rcp), Mg = pk2(kRoundMagic, kRoundMagic);
    const uint64_t v01 = pk2(v.x, v.y), v23 = pk2(v.z, v.w);
    const uint64_t y01 = fma2(v01, R, Mg), y23 = fma2(v23, R, Mg);
    const uint64_t d01 = fma2(v01, R, sub2(Mg, y01)), d23 = fma2(v23, R, sub2(Mg, y23));
    float y0, y1, y2, y3, d0, d1, d2, d3;
    upk2(y01, y0, y1);
    upk2(y23, y2, y3);
    upk2(d01, d0, d1);
    upk2(d23, d2, d3);
    const uint32_t lo01 = __byte_perm(__float_as_uint(y0), __float_as_uint(y1), 0x0040);
    const uint32_t lo23 = __byte_perm(__float_as_uint(y2), __float_as_uint(y3), 0x0040);
    dmax = fmaxf(fmaxf(fabsf(d0), fabsf(d1)), fmaxf(fabsf(d2), fabsf(d3)));
    return __byte_perm(lo01, lo23, 0x5410);
}

// Sixteen codes from four float4: one tie check (one branch) for all of them,
// so the four independent chains interleave.
__device__ __forceinline__ uint4 pack16(const float4& a, const float4& b, const float4& c, const float4& d,
                                        const ScaleInfo& si) {
    float m0, m1, m2, m3;
    uint4 w;
    w.x = pack4_fast(a, si.rcp, m0);
    w.y = pack4_fast(b, si.rcp, m1);
    w.z = pack4_fast(c, si.rcp, m2);
    w.w = pack4_fast(d, si.rcp, m3);
    if (!si.fast || fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) > kTieGuardFma) {
        if (!si.fast || m0 > kTieGuardFma) w.x = pack4_repair(a, w.x, si.scale, si.rcp, si.fast);
        if (!si.fast || m1 > kTieGuardFma) w.y = pack4_repair(b, w.y, si.scale, si.rcp, si.fast);
        if (!si.fast || m2 > kTieGuardFma) w.z = pack4_repair(c, w.z, si.scale, si.rcp, si.fast);
        if (!si.fast || m3 > kTieGuardFma) w.w = pack4_repair(d, w.w, si.scale, si.rcp, si.fast);
    }
    return w;
}

// Four codes packed little-endian into one word: three fp32 operations per
// element and one tie check per four; a word with a near-tie element is
// repaired per element.
__device__ __forceinline__ uint32_t pack4(const float4& v, const ScaleInfo& si) {
    float dm;
    const uint32_t w = pack4_fast(v, si.rcp, dm);
    if (si.fast && dm <= kTieGuardFma) return w;
    return pack4_repair(v, w, si.scale, si.rcp, si.fast);
}

}  // namespace kz
