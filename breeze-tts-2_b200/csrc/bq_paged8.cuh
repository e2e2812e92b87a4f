// Shared pieces of the 8-bit paged KV cache (bq_paged8_*): scales, and e4m3 codes
// to and from fp32 and f16.
//
// A cache entry is code * 2^e, e4m3 codes and one e for each block of positions and
// kv head. A power of two, since a block grows token by token: when a later token
// needs a larger scale, dividing the codes that are there by a power of two is exact
// (codes that become subnormal aside), and e4m3 has its four significant bits at any
// scale, so the quotient largest / 448 would gain nothing.
#pragma once

#include "bq_paged.cuh"

namespace bq {

// Exponents are from -60 to 60: products of two powers of two of the cache, and
// sums relative to the largest of them, stay far inside fp32's range.
constexpr int kExpMost = 60, kExpBias = 127;

struct Paged8Scales {
    void* k;
    int64_t ks_page, ks_head;
    void* v;
    int64_t vs_page, vs_head;
    int32_t block_shift;  // slot >> block_shift: the slot's block in its page
};

__device__ __forceinline__ int scale_exp(uint32_t byte) { return min(max(int(byte) - kExpBias, -kExpMost), kExpMost); }
// 2^e, exactly, for e from -126 to 127.
__device__ __forceinline__ float exp_scale(int e) { return __int_as_float((e + 127) << 23); }
// The scale byte of head j, block `blk` of a page.
__device__ __forceinline__ const uint8_t* k_scale(const Paged8Scales& s, int page, int j, int blk) {
    return static_cast<const uint8_t*>(s.k) + page * s.ks_page + j * s.ks_head + blk;
}
__device__ __forceinline__ const uint8_t* v_scale(const Paged8Scales& s, int page, int j, int blk) {
    return static_cast<const uint8_t*>(s.v) + page * s.vs_page + j * s.vs_head + blk;
}

// The exponent of a part's sum of exponentials l goes into its reference m, as far as fp32 holds the two together (a
// reference of 2^24 and more does not take every integer: equal parts would be weighed by up to a factor of two each),
// and out of l; returns what the part's outputs are to be multiplied with.
__device__ __forceinline__ float settle_part(float& m, float& l) {
    if (!(l > 0.f && l < INFINITY)) return 1.f;
    const float to = m + float(int(__float_as_uint(l) >> 23) - 127), f = ex2(m - to);
    m = to;
    l *= f;
    return f;
}

// Four codes -> two pairs of f16 (exact; NaN stays NaN).
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = e4m3x2_to_f16x2(uint16_t(w));
    hi = e4m3x2_to_f16x2(uint16_t(w >> 16));
}
__device__ __forceinline__ void codes_f32(uint32_t w, float (&v)[4]) {
    uint32_t lo, hi;
    codes_f16(w, lo, hi);
    unpack2<__half>(lo, v[0], v[1]);
    unpack2<__half>(hi, v[2], v[3]);
}
// Two values -> codes, to nearest even, at most 448; a in the low byte. NaN -> NaN.
__device__ __forceinline__ uint32_t f32_codes(float a, float b) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(b), "f"(a));
    return d;
}

}  // namespace bq
