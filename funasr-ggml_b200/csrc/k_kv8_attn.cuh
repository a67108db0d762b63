// What decode (k_kv8_attention.cu) and prefill attention (k_kv8_prefill.cu) over the 8-bit
// page pool share. Row m attends to tokens t in [0, pos[m]] of its sequence; query head H uses
// KV head H / (n_heads / n_kv_heads):
//   s_t = dk_t (q . kq_t),  o = sum_t exp(s_t - max s) dv_t vq_t / sum_t exp(s_t - max s)
// with kq, vq the stored 8-bit values and dk, dv the scales of their vectors. The scales
// multiply a score and a weight, never the 128 values.
#pragma once

#include "k_kv8.cuh"
#include "tc_common.cuh"
#include "funasr_dec.h"

#include <cmath>
#include <string>

namespace fa {

int report_op_error(int code, const char* msg);   // fa_api.cu
int ensure_device_configured();                   // fa_api.cu: kernel attributes of the current device, once

namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;

struct Kv8AttnArgs {
    const float* q;          // [M][Hq][128], pre-scaled
    int M, Hq, Hkv;
    const int* pos;
    const int* slot;
    const int* block_table;
    int bt_stride;
    int n_pages;
    const unsigned char* pool;   // one layer
    const int2* tiles;       // prefill: (first row, rows)
    int n_tiles;
    __half* out16;
    __half* out16_lo;
    float* out32;
    int* err;
};

// A row that cannot be served.
__device__ __forceinline__ bool row_bad(const Kv8AttnArgs& a, int m) {
    const int pos = a.pos[m], slot = a.slot[m];      // both under way at once
    return pos < -1 || pos / kPageTokens >= a.bt_stride || (pos >= 0 && slot < 0);
}

// The power of two at or below x, within 2^-126 .. 2^126, and the inverse of such a one.
__device__ __forceinline__ float pow2_floor(float x) {
    return __uint_as_float(min(max(__float_as_uint(x) & 0x7f800000u, 0x00800000u), 0x7e800000u));
}
__device__ __forceinline__ float pow2_inverse(float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); }

// 2^x, results below 2^-126 as zero: weights of a softmax.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// N consecutive outputs from offset o, a multiple of 4.
template <int N>
__device__ __forceinline__ void store_values(const Kv8AttnArgs& a, size_t o, const float (&v)[N]) {
    if (a.out32) {
#pragma unroll
        for (int k = 0; k < N; k += 4)
            *reinterpret_cast<float4*>(a.out32 + o + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    }
    if (a.out16) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const __half2 h = __floats2half2_rn(v[k + 2 * e], v[k + 2 * e + 1]);
                const float2 f = __half22float2(h);
                const __half2 r = __floats2half2_rn(__fsub_rn(v[k + 2 * e], f.x), __fsub_rn(v[k + 2 * e + 1], f.y));
                hi[e] = *reinterpret_cast<const uint32_t*>(&h);
                lo[e] = *reinterpret_cast<const uint32_t*>(&r);
            }
            *reinterpret_cast<uint2*>(a.out16 + o + k) = make_uint2(hi[0], hi[1]);
            if (a.out16_lo) *reinterpret_cast<uint2*>(a.out16_lo + o + k) = make_uint2(lo[0], lo[1]);
        }
    }
}
// The outputs x / l: 0 where no token takes part (l = 0).
template <int N>
__device__ __forceinline__ void store_quotients(const Kv8AttnArgs& a, size_t o, const float (&x)[N], float l) {
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = l == 0.0f ? 0.0f : x[k] / l;
    store_values<N>(a, o, v);
}
__device__ __forceinline__ void store16(const Kv8AttnArgs& a, size_t o, const float (&x)[16], float l) {
    store_quotients<16>(a, o, x, l);
}
__device__ __forceinline__ void store4(const Kv8AttnArgs& a, size_t o, float4 x, float l) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    store_quotients<4>(a, o, v, l);
}

}  // namespace kv8

// The arguments that decode and prefill share, checked; FA_OK or the recorded error.
int kv8_attention_check(const char* what, const kv8::Kv8AttnArgs& a, int format, const void* scratch,
                        size_t scratch_bytes, size_t need);
// The pool as rows of 128 bytes (33 a tile: 16 of K, 16 of V, the scales); a box is K and V.
bool make_kv8_tile_map(CUtensorMap* tm, const void* pool, long long rows);

}  // namespace fa
