// The 8-bit page pool: layout, the quantiser and the expansion shared by its kernels.
//
// One page of one layer holds 16 tokens of a sequence for every KV head, as the f16 pool's
// page does, in kv_heads tiles of 4224 bytes:
//   [K 16 tokens x 128][V 16 tokens x 128][K scales 16 x f32][V scales 16 x f32]
// 4224 = 33 x 128, so a head's tile is one aligned bulk copy. Pool: [layer][page][kv head][tile].
//
// A 128-value vector x (one token, one KV head, K or V) is stored as a scale d and x / d:
//   int8  d = max(amax / 127, 2^-126) rounded to f32, x / d rounded to the nearest integer,
//         ties to even: |error| <= d / 2
//   e4m3  d = the smallest power of two >= 2^-126 with amax <= 448 d, x / d (exact) rounded
//         to e4m3, ties to even
// A vector that holds a NaN or an infinity gets d = NaN and zeros: it reads back as NaN.
// The scale belongs to one token: a block of more tokens would have to be requantised
// whenever a later token is larger, so its bytes would depend on how the tokens were cut
// into calls, and every decode step would rewrite a page; it would save 3 % of the bytes.
#pragma once

#include "fa_kernels.cuh"

#include <cuda_fp8.h>

namespace fa {
namespace kv8 {

constexpr int D = 128;
constexpr int kTileBytes = 4224;
constexpr int kPartBytes = kPageTokens * D;        // K or V of one tile
constexpr int kScaleOff = 2 * kPartBytes;          // 16 K scales, then 16 V scales
constexpr float kMinScale = 1.17549435e-38f;       // 2^-126
constexpr int kInt8 = 0, kE4m3 = 1;

// The scale of a vector whose largest |x| has these bits (an infinity or NaN: NaN).
template <int FMT>
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
    if (FMT == kInt8) return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 127.0f), kMinScale);
    // amax = 1.f x 2^e <= 448 d = 1.75 x 2^8 d
    const int e = (int)(amax_bits >> 23);
    const int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
    return __uint_as_float((uint32_t)max(k, 1) << 23);
}

// x / d rounded to the nearest integer, ties to even, exactly, as the low byte of the result.
// m = 1.5 * 2^23 + x * inv rounds the product to an integer that is off by less than one from
// the quotient; its remainder r = x - q d is exact in f32 (x and q d are multiples of the
// smaller of their last places and nearly cancel), so comparing |r| with d / 2 settles on which
// side of the border x / d lies. border collects the largest |r|: only where that reaches d / 2
// does a value need settle().
constexpr float kRoundMagic = 12582912.0f;         // 1.5 * 2^23: an even integer, low byte 0
__device__ __forceinline__ uint32_t round_quotient(float x, float d, float inv, float& border) {
    const float m = __fmaf_rn(x, inv, kRoundMagic);
    border = fmaxf(border, fabsf(__fmaf_rn(-__fsub_rn(m, kRoundMagic), d, x)));
    return __float_as_uint(m);
}
__device__ __forceinline__ uint32_t settle(uint32_t m, float x, float d) {
    const float r = __fmaf_rn(-__fsub_rn(__uint_as_float(m), kRoundMagic), d, x), a = fabsf(r), h = 0.5f * d;
    return a > h || (a == h && (m & 1)) ? m + (r > 0.0f ? 1u : ~0u) : m;
}

__device__ __forceinline__ uint32_t join4(const uint32_t (&m)[4]) {      // low bytes
    return __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
}

// Four values of a vector with scale d as stored bytes. inv = 1 / d (for e4m3 exact).
template <int FMT>
__device__ __forceinline__ uint32_t pack4(const float* x, float d, float inv) {
    if (FMT == kInt8) {
        uint32_t m[4];
        float border = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = round_quotient(x[k], d, inv, border);
        if (border >= 0.5f * d) {
#pragma unroll
            for (int k = 0; k < 4; ++k) m[k] = settle(m[k], x[k], d);
        }
        return join4(m);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Two f16 pairs (exact) of the four stored values of a word, in order. int8: the byte
// offset by 128 under the exponent of 1024 is 1152 + value.
template <int FMT>
__device__ __forceinline__ void expand4(uint32_t w, __half2& a, __half2& b) {
    if (FMT == kInt8) {
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
        a = __hsub2(*reinterpret_cast<const __half2*>(&lo), off);
        b = __hsub2(*reinterpret_cast<const __half2*>(&hi), off);
    } else {
        a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3));
        b = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
    }
}

}  // namespace kv8
}  // namespace fa
