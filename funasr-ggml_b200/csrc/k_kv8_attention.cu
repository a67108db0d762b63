// Attention over the 8-bit page pool (k_kv8.cuh): decode rows and causal prefill tiles.
//
// Row m attends to tokens t in [0, pos[m]] of its sequence; query head H uses KV head
// H / (n_heads / n_kv_heads):
//   s_t = dk_t (q . kq_t),  o = sum_t exp(s_t - max s) dv_t vq_t / sum_t exp(s_t - max s)
// with kq, vq the stored 8-bit values and dk, dv the scales of their vectors. The scales
// multiply a score and a weight, never the 128 values.
#include "k_kv8.cuh"
#include "funasr_dec.h"

#include <cmath>
#include <string>

namespace fa {

int report_op_error(int code, const char* msg);   // fa_api.cu

namespace {

using namespace kv8;

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

__device__ __forceinline__ void store_out(const Kv8AttnArgs& a, size_t o, float v) {
    if (a.out16) {
        const __half h = __float2half_rn(v);
        a.out16[o] = h;
        if (a.out16_lo) a.out16_lo[o] = __float2half_rn(__fsub_rn(v, __half2float(h)));
    }
    if (a.out32) a.out32[o] = v;
}

// One query vector of one row by a warp, lane l holding dims 4l .. 4l+3.
template <int FMT>
__device__ void attend_row(const Kv8AttnArgs& a, int m, int H, int lane) {
    const int pos = a.pos[m];
    const size_t o = ((size_t)m * a.Hq + H) * D + 4 * lane;
    if (pos < -1 || pos / kPageTokens >= a.bt_stride || (pos >= 0 && a.slot[m] < 0)) {
        if (lane == 0 && H == 0) record_error(a.err, kDevErrBadLen);
        return;
    }
    const int h = H / (a.Hq / a.Hkv);
    const float4 q = *reinterpret_cast<const float4*>(a.q + o);
    float mx = -INFINITY, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p * kPageTokens <= pos; ++p) {
        const int page = a.block_table[(size_t)a.slot[m] * a.bt_stride + p];
        if (page < 0 || page >= a.n_pages) {
            if (lane == 0) record_error(a.err, kDevErrBadPage);
            continue;
        }
        const unsigned char* tile = a.pool + ((size_t)page * a.Hkv + h) * kTileBytes;
        const float* scale = reinterpret_cast<const float*>(tile + kScaleOff);
        const int n = min(kPageTokens, pos + 1 - p * kPageTokens);
        for (int t = 0; t < n; ++t) {
            __half2 x, y;
            expand4<FMT>(*reinterpret_cast<const uint32_t*>(tile + t * D + 4 * lane), x, y);
            const float2 k0 = __half22float2(x), k1 = __half22float2(y);
            float s = q.x * k0.x + q.y * k0.y + q.z * k1.x + q.w * k1.y;
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
            s *= scale[t] * kLog2e;
            const float top = fmaxf(mx, s);
            const float alpha = exp2f(mx - top), w = exp2f(s - top);
            mx = top;
            sum = sum * alpha + w;
            expand4<FMT>(*reinterpret_cast<const uint32_t*>(tile + kPartBytes + t * D + 4 * lane), x, y);
            const float2 v0 = __half22float2(x), v1 = __half22float2(y);
            const float wv = w * scale[kPageTokens + t];
            acc[0] = acc[0] * alpha + wv * v0.x;
            acc[1] = acc[1] * alpha + wv * v0.y;
            acc[2] = acc[2] * alpha + wv * v1.x;
            acc[3] = acc[3] * alpha + wv * v1.y;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) store_out(a, o + i, sum == 0.0f ? 0.0f : acc[i] / sum);
}

template <int FMT>
__global__ void __launch_bounds__(128) kv8_decode_kernel(Kv8AttnArgs a) {
    const int H = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (H < a.Hq) attend_row<FMT>(a, blockIdx.x, H, threadIdx.x & 31);
}

template <int FMT>
__global__ void __launch_bounds__(128) kv8_prefill_kernel(Kv8AttnArgs a) {
    const int2 tile = a.tiles[blockIdx.x];
    if (tile.x < 0 || tile.y < 1 || tile.y > 128 / (a.Hq / a.Hkv) || tile.x > a.M - tile.y) {
        if (blockIdx.y == 0 && threadIdx.x == 0) record_error(a.err, kDevErrBadPos);
        return;
    }
    const int H = blockIdx.y;
    for (int r = threadIdx.x >> 5; r < tile.y; r += 4) attend_row<FMT>(a, tile.x + r, H, threadIdx.x & 31);
}

bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// The arguments that decode and prefill share, checked; FA_OK or the recorded error.
int check(const std::string& what, const Kv8AttnArgs& a, int format, const void* scratch, size_t scratch_bytes,
          size_t need) {
    if (!a.q || !a.pos || !a.slot || !a.block_table || !a.pool || (!a.out16 && !a.out32) || a.M <= 0 || a.Hq <= 0 ||
        a.Hkv <= 0 || a.bt_stride <= 0 || a.n_pages <= 0)
        return report_op_error(FA_ERR_INVALID_ARG, (what + ": null or non-positive argument").c_str());
    if (a.out16_lo && !a.out16)
        return report_op_error(FA_ERR_INVALID_ARG, (what + ": out16_lo needs out16").c_str());
    if (format != FA_KV8_INT8 && format != FA_KV8_E4M3)
        return report_op_error(FA_ERR_INVALID_ARG, (what + ": unknown format").c_str());
    if (a.Hq % a.Hkv || a.Hq / a.Hkv > 8)
        return report_op_error(FA_ERR_INVALID_ARG,
                               (what + ": n_heads must be 1 to 8 times n_kv_heads").c_str());
    if (misaligned(a.q, 16) || misaligned(a.pool, 128) || misaligned(a.out16, 16) || misaligned(a.out16_lo, 16) ||
        misaligned(a.out32, 16) || misaligned(scratch, 16))
        return report_op_error(FA_ERR_INVALID_ARG,
                               (what + ": q, outputs and scratch must be 16-byte, pool 128-byte aligned").c_str());
    if (a.Hq > 65535 || (long long)a.bt_stride * kPageTokens > 0x7fffffffll)
        return report_op_error(FA_ERR_CAPACITY, (what + ": n_heads or bt_stride too large").c_str());
    if (need && (!scratch || scratch_bytes < need))
        return report_op_error(FA_ERR_INVALID_ARG, (what + ": scratch of " + std::to_string(need) +
                                                    " bytes required").c_str());
    return FA_OK;
}

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return FA_OK;
    return report_op_error(FA_ERR_CUDA, (std::string(what) + ": " + cudaGetErrorString(e)).c_str());
}

}  // namespace
}  // namespace fa

extern "C" FA_API size_t fa_op_attention_kv8_scratch_bytes(int M, int n_heads, int n_kv_heads) {
    return M > 0 && n_heads > 0 && n_kv_heads > 0 ? 16 : 0;
}

extern "C" FA_API size_t fa_op_prefill_attention_kv8_scratch_bytes(int n_tiles, int n_heads, int n_kv_heads) {
    return n_tiles > 0 && n_heads > 0 && n_kv_heads > 0 ? 16 : 0;
}

extern "C" FA_API int fa_op_paged_attention_kv8(const float* q, int M, int n_heads, int n_kv_heads, const int* pos,
                                                const int* slot, const int* bt, int bt_stride, int n_pages,
                                                int format, const void* pool_layer, void* scratch,
                                                size_t scratch_bytes, uint16_t* out16, uint16_t* out16_lo,
                                                float* out32, int* err, void* stream) {
    using namespace fa;
    Kv8AttnArgs a{q, M, n_heads, n_kv_heads, pos, slot, bt, bt_stride, n_pages,
                  static_cast<const unsigned char*>(pool_layer), nullptr, 0, reinterpret_cast<__half*>(out16),
                  reinterpret_cast<__half*>(out16_lo), out32, err};
    if (int rc = check("fa_op_paged_attention_kv8", a, format, scratch, scratch_bytes,
                       fa_op_attention_kv8_scratch_bytes(M, n_heads, n_kv_heads)))
        return rc;
    const dim3 grid(M, (n_heads + 3) / 4);
    if (format == FA_KV8_INT8) kv8_decode_kernel<kInt8><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    else kv8_decode_kernel<kE4m3><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    return launched("fa_op_paged_attention_kv8");
}

extern "C" FA_API int fa_op_prefill_attention_kv8(const float* q, int M, int n_heads, int n_kv_heads, const int* pos,
                                                  const int* slot, const int* bt, int bt_stride, int n_pages,
                                                  int format, const void* pool_layer, const int* tiles, int n_tiles,
                                                  void* scratch, size_t scratch_bytes, uint16_t* out16,
                                                  uint16_t* out16_lo, float* out32, int* err, void* stream) {
    using namespace fa;
    Kv8AttnArgs a{q, M, n_heads, n_kv_heads, pos, slot, bt, bt_stride, n_pages,
                  static_cast<const unsigned char*>(pool_layer), reinterpret_cast<const int2*>(tiles), n_tiles,
                  reinterpret_cast<__half*>(out16), reinterpret_cast<__half*>(out16_lo), out32, err};
    if (!tiles || n_tiles <= 0 || misaligned(tiles, 8))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_prefill_attention_kv8: tiles missing or not 8-byte aligned");
    if (int rc = check("fa_op_prefill_attention_kv8", a, format, scratch, scratch_bytes,
                       fa_op_prefill_attention_kv8_scratch_bytes(n_tiles, n_heads, n_kv_heads)))
        return rc;
    const dim3 grid(n_tiles, n_heads);
    if (format == FA_KV8_INT8) kv8_prefill_kernel<kInt8><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    else kv8_prefill_kernel<kE4m3><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    return launched("fa_op_prefill_attention_kv8");
}
