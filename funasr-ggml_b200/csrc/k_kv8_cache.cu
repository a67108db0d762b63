// Writing the 8-bit page pool (k_kv8.cuh) and reading it back: the raw append, kernel (1)
// with an 8-bit end (per-head Q/K RMSNorm + NEOX RoPE + append), and the gather into
// head-major slabs. The f16 pool's forms of the three are in k_append.cu.
//
// All three are bound by HBM: a vector costs 132 bytes in the pool against its 256 (f16) or
// 512 (f32) outside. Measured (a copy reaches 6.54 TB/s): append of 4,432 f32 tokens x 8 layers
// x 8 heads 58.7 us, 6.2 TB/s; read-back of 4001 tokens x 28 layers to bf16 107 us, 6.5 TB/s.
#include "k_append.cuh"
#include "k_kv8.cuh"
#include "funasr_dec.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <string>

namespace fa {

int report_op_error(int code, const char* msg);   // fa_api.cu

namespace {

using namespace kv8;

// Where a row's token goes: its page, or -1 (padding, or an error that is flagged once).
__device__ __forceinline__ int token_page(const int* bt, int bt_stride, int n_pages, int slot, int pos, int* err,
                                          bool flag) {
    if (pos == -1) return -1;
    if (pos < 0 || pos / kPageTokens >= bt_stride || slot < 0) {
        if (flag) record_error(err, kDevErrBadPos);
        return -1;
    }
    const int page = bt[(size_t)slot * bt_stride + pos / kPageTokens];
    if (page < 0 || page >= n_pages) {
        if (flag) record_error(err, kDevErrBadPage);
        return -1;
    }
    return page;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = h2_to_f2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

struct Kv8AppendArgs {
    const void* k;           // [M] rows of [n_layers][Hkv][128], row_stride elements apart
    const void* v;
    long long row_stride;
    int M, n_layers, Hkv;
    const int* pos;
    const int* slot;
    const int* block_table;
    int bt_stride;
    int n_pages;
    unsigned char* pool;
    int* err;
};

// Raw append: a warp per P (layer, KV head) pairs of a row, its half-warps the K and the V
// vector of a pair, a lane 8 consecutive values of each; the loads of all pairs are under way
// before the row's place in the pool is looked up. The pairs' largest magnitudes are reduced
// over the half-warp together (each exchange halves the pairs a lane carries), so that the
// scales and their reciprocals are computed once, side by side, and handed back.
template <int FMT, typename T, int P>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8AppendArgs a, unsigned blocks_per_row) {
    static_assert(P == 1 || P == 4, "the exchanges below");
    const int m = blockIdx.x / blocks_per_row;
    const int i0 = (int)((blockIdx.x - m * blocks_per_row) * 8 + (threadIdx.x >> 5)) * P;
    const int lane = threadIdx.x & 31, part = lane >> 4, c = lane & 15;
    const int n_pairs = a.n_layers * a.Hkv;
    if (i0 >= n_pairs) return;
    const T* src = reinterpret_cast<const T*>(part ? a.v : a.k) + (size_t)m * a.row_stride + 8 * c;
    float x[P][8];
#pragma unroll
    for (int u = 0; u < P; ++u) load8(src + (size_t)min(i0 + u, n_pairs - 1) * D, x[u]);
    const int pos = a.pos[m];
    const int page = token_page(a.block_table, a.bt_stride, a.n_pages, a.slot[m], pos, a.err, lane == 0);
    if (page < 0) return;
    uint32_t amax[P];
#pragma unroll
    for (int u = 0; u < P; ++u) {
        amax[u] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax[u] = max(amax[u], __float_as_uint(x[u][i]) & 0x7fffffffu);
    }
    uint32_t top = amax[0];
    if (P == 4) {                                      // lane c ends with pair c / 4
        uint32_t two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t keep = (c & 8) ? amax[(i + 2) % P] : amax[i % P];
            const uint32_t send = (c & 8) ? amax[i % P] : amax[(i + 2) % P];
            two[i] = max(keep, __shfl_xor_sync(0xffffffffu, send, 8));
        }
        const uint32_t keep = (c & 4) ? two[1] : two[0], send = (c & 4) ? two[0] : two[1];
        top = max(keep, __shfl_xor_sync(0xffffffffu, send, 4));
    } else {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 4));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const float d_mine = scale_of<FMT>(top), inv_mine = __frcp_rn(d_mine);
    const int t = pos % kPageTokens;
    int l = i0 / a.Hkv, h = i0 - l * a.Hkv;
#pragma unroll
    for (int u = 0; u < P; ++u) {
        const float d = P == 1 ? d_mine : __shfl_sync(0xffffffffu, d_mine, (lane & 16) + 4 * u);
        const float inv = P == 1 ? inv_mine : __shfl_sync(0xffffffffu, inv_mine, (lane & 16) + 4 * u);
        if (i0 + u < n_pairs) {
            uint2 q = make_uint2(0, 0);
            if (d == d) q = make_uint2(pack4<FMT>(x[u], d, inv), pack4<FMT>(x[u] + 4, d, inv));
            unsigned char* tile = a.pool + (((size_t)l * a.n_pages + page) * a.Hkv + h) * kTileBytes;
            *reinterpret_cast<uint2*>(tile + part * kPartBytes + t * D + 8 * c) = q;
            if (c == 0) reinterpret_cast<float*>(tile + kScaleOff)[part * kPageTokens + t] = d;
        }
        if (++h == a.Hkv) {
            h = 0;
            ++l;
        }
    }
}

// Warps of a CTA: 4096 rows of 32 head vectors took 27.4 us with 8, 22.7 with 4, 22.2 with 2 and
// 22.9 with 1, before keys were rounded exactly (a CTA's registers are free again only when its slowest warp ends).
constexpr int kQkvWarps = 2;

struct Kv8QkvArgs {
    const float* qkv;        // [M][(Hq + 2 Hkv) * 128]
    int M, Hq, Hkv;
    const int* pos;
    const int* slot;
    const int* block_table;
    int bt_stride;
    int n_pages;
    const float* qn_w;
    const float* kn_w;
    float eps, q_scale;
    const float2* rope;      // [max_pos][64]
    int max_pos;
    unsigned char* pool;     // one layer
    float* q_out;            // [M][Hq][128]
    int* err;
};

__device__ __forceinline__ void load4(const float* vec, int lane, float (&x)[4]) {
    const float2 a = reinterpret_cast<const float2*>(vec)[lane], b = reinterpret_cast<const float2*>(vec)[lane + 32];
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
}

// K is stored as if it had been computed in 64 bits and rounded once. Its f32 values are off by
// less than 11 x 2^-24 of the vector's largest (the norm's scale by 3.5 roundings, two products
// and a rotation by 4, whose terms together reach sqrt(2) of it), so their bytes can differ from
// those of the exact values only next to a border: where one lies within that distance (for int8
// twice that and an ulp, since the scale is off by as much), the vector is computed again in 64
// bits, a few vectors in a hundred. So is one whose f32 values are not known that well: where a
// square, their mean, a product or a rotation may have left f32's normal range.
template <int FMT>
constexpr float kKeyError = (FMT == kInt8 ? 23.5f : 12.5f) / (1 << 24);
// Mean square and epsilon within 2^-120 .. 2^120: squares that are lost below 2^-149 then weigh
// less than 2^-28 of the mean, and none of 128 reached 2^128.
__device__ __forceinline__ bool norm_in_range(float scale) { return scale >= 0x1p-60f && scale <= 0x1p60f; }
// The last place of a subnormal is 2^-49 of such a vector's largest, or less; that of a normalised
// value is so once more, and then multiplied by a weight of at most w_max.
__device__ __forceinline__ bool key_in_range(float amax) { return amax >= 0x1p-100f && amax <= FLT_MAX; }
__device__ __forceinline__ bool weights_in_range(float w_max, float e) { return w_max <= e * 0x1p120f; }

// pack4 of key values, unless a value that differs by e may round otherwise (near).
template <int FMT>
__device__ __forceinline__ uint32_t pack_key(const float (&x)[4], float d, float inv, float e, bool& near) {
    if (FMT == kInt8) {
        uint32_t m[4];
        float border = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = round_quotient(x[k], d, inv, border);
        near = border >= 0.5f * d - e;
        return join4(m);
    }
    const float a[4] = {x[0] - e, x[1] - e, x[2] - e, x[3] - e}, b[4] = {x[0] + e, x[1] + e, x[2] + e, x[3] + e};
    const uint32_t q = pack4<FMT>(a, d, inv);
    near = q != pack4<FMT>(b, d, inv);
    return q;
}

// A key vector in 64 bits, by a warp: the lane's four stored bytes, and the scale. A value that is
// past f32's range counts as infinite.
template <int FMT>
__device__ __noinline__ uint32_t exact_key(const float* vec, int lane, const float* w, const float2* rot, float eps,
                                           float& d) {
    const float2 lo = reinterpret_cast<const float2*>(vec)[lane], hi = reinterpret_cast<const float2*>(vec)[lane + 32];
    double y[4] = {lo.x, lo.y, hi.x, hi.y};
    double ss = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const double scale = rsqrt(ss * (1.0 / D) + (double)eps);
    double amax = 0.0;
    bool finite = true;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] *= scale * (double)w[k];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const double a = y[k], b = y[k + 2], c = rot[k].x, s = rot[k].y;
        y[k] = a * c - b * s;
        y[k + 2] = a * s + b * c;
        amax = fmax(amax, fmax(fabs(y[k]), fabs(y[k + 2])));
        finite = finite && fabs(y[k]) <= FLT_MAX && fabs(y[k + 2]) <= FLT_MAX;
    }
    uint32_t q = 0;
    if (!__all_sync(0xffffffffu, finite)) {
        d = __uint_as_float(0x7fffffffu);
        return q;
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (FMT == kInt8) {
        d = fmaxf(__double2float_rn(amax / 127.0), kMinScale);
        const double inv = 1.0 / (double)d;
#pragma unroll
        for (int k = 0; k < 4; ++k) q |= ((uint32_t)__double2int_rn(y[k] * inv) & 0xffu) << (8 * k);
        return q;
    }
    d = scale_of<FMT>(__float_as_uint(__double2float_ru(amax)));   // at most 448 d, and so rounded up
    const double inv = (double)__frcp_rn(d);                      // exact: a power of two
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {                                  // towards zero with the rest kept in the last bit
        const double v = y[k] * inv;
        const float z = __double2float_rz(v);
        f[k] = (double)z == v ? z : __uint_as_float(__float_as_uint(z) | 1u);
    }
    return pack4<FMT>(f, 1.0f, 1.0f);
}

// Kernel (1) with an 8-bit end: a CTA per row and kQkvWarps * V of its head vectors, a warp V of
// them (lane l holding dims 2l, 2l+1, 64+2l, 65+2l: both rotation pairs of a lane stay in it),
// whose loads are under way together with that of the row's position. With V = 4 the vectors'
// sums of squares are reduced over the warp together: each exchange halves the vectors a lane
// carries, and the norms' square root and division, and the scales and reciprocals, are computed
// once, side by side.
// Bound: issue (2.6 instructions a cycle, 140 a vector) and HBM. 4096 rows of 32 vectors (111 MB)
// take 27.1 us, 4.1 TB/s; 26.5 without the checks of the keys' range, 22.2 with keys rounded from
// their f32 values.
template <int FMT, int V>
__global__ void __launch_bounds__(kQkvWarps * 32) kv8_qkv_kernel(Kv8QkvArgs a) {
    static_assert(V == 1 || V == 4, "the exchanges below");
    const int m = blockIdx.x;
    const int lane = threadIdx.x & 31;
    const int j0 = blockIdx.y * kQkvWarps * V + (threadIdx.x >> 5);
    const int n_vec = a.Hq + 2 * a.Hkv;
    if (j0 >= n_vec) return;
    float x[V][4];
#pragma unroll
    for (int u = 0; u < V; ++u) {
        load4(a.qkv + ((size_t)m * n_vec + min(j0 + kQkvWarps * u, n_vec - 1)) * D, lane, x[u]);
    }
    float qw[4], kw[4];
    load4(a.qn_w, lane, qw);
    load4(a.kn_w, lane, kw);
    const int pos = a.pos[m];
    if (pos == -1) return;
    if (pos < 0 || pos >= a.max_pos) {
        if (lane == 0) record_error(a.err, kDevErrBadPos);
        return;
    }
    const float4 cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * (D / 2))[lane];
    const float2 rot[2] = {make_float2(cs.x, cs.y), make_float2(cs.z, cs.w)};
    const bool stores = j0 + kQkvWarps * (V - 1) >= a.Hq;                 // a K or V head among the warp's
    const int page =
        stores ? token_page(a.block_table, a.bt_stride, a.n_pages, a.slot[m], pos, a.err, lane == 0) : -1;
    float scale[V];
    uint32_t far;                                                 // bit 8 u: not norm_in_range
    if (V == 4) {
        double two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const double lo = norm_squares(x[i % V]), hi = norm_squares(x[(i + 2) % V]);
            two[i] = ((lane & 16) ? hi : lo) + __shfl_xor_sync(0xffffffffu, (lane & 16) ? lo : hi, 16);
        }
        double ss = ((lane & 8) ? two[1] : two[0]) + __shfl_xor_sync(0xffffffffu, (lane & 8) ? two[0] : two[1], 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float mine = norm_scale(ss, a.eps);                 // lane l: vector l / 8
        far = __ballot_sync(0xffffffffu, !norm_in_range(mine));
#pragma unroll
        for (int u = 0; u < V; ++u) scale[u] = __shfl_sync(0xffffffffu, mine, 8 * u);
    } else {
        double ss = norm_squares(x[0]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        scale[0] = norm_scale(ss, a.eps);
        far = !norm_in_range(scale[0]);
    }
    uint32_t top = 0;                                             // lane l: of the warp's stored vector l % V
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const int j = j0 + kQkvWarps * u;
        if (j >= n_vec) break;
        if (j < a.Hq) {
            norm_rope_apply(qw, rot, scale[u], x[u]);
            float2* dst = reinterpret_cast<float2*>(a.q_out + ((size_t)m * a.Hq + j) * D) + lane;
            dst[0] = make_float2(__fmul_rn(x[u][0], a.q_scale), __fmul_rn(x[u][1], a.q_scale));
            dst[32] = make_float2(__fmul_rn(x[u][2], a.q_scale), __fmul_rn(x[u][3], a.q_scale));
        } else {
            if (j < a.Hq + a.Hkv) norm_rope_apply(kw, rot, scale[u], x[u]);
            uint32_t amax = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = max(amax, __float_as_uint(x[u][k]) & 0x7fffffffu);
            amax = __reduce_max_sync(0xffffffffu, amax);
            if (lane % V == u) top = amax;
        }
    }
    if (page < 0) return;
    const float d_mine = scale_of<FMT>(top), inv_mine = __frcp_rn(d_mine);
    const float amax_mine = __uint_as_float(top), e_mine = amax_mine * kKeyError<FMT>;
    // keys out of range, and e4m3 scales that the error of the largest value may change
    const bool other_scale = FMT != kInt8 && scale_of<FMT>(__float_as_uint(amax_mine + e_mine)) !=
                                                 scale_of<FMT>(__float_as_uint(amax_mine - e_mine));
    const uint32_t unsure = __ballot_sync(0xffffffffu, !key_in_range(amax_mine) || other_scale);
    const float w_max = fmaxf(fmaxf(fabsf(kw[0]), fabsf(kw[1])), fmaxf(fabsf(kw[2]), fabsf(kw[3])));   // the lane's
    const int t = pos % kPageTokens;
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const int j = j0 + kQkvWarps * u;
        if (j < a.Hq) continue;
        if (j >= n_vec) break;
        const int part = j < a.Hq + a.Hkv ? 0 : 1, h = j - a.Hq - part * a.Hkv;
        float d = __shfl_sync(0xffffffffu, d_mine, u);
        const float inv = __shfl_sync(0xffffffffu, inv_mine, u);
        uint32_t q = 0;
        if (part == 0) {
            bool near;
            const float e = __shfl_sync(0xffffffffu, e_mine, u);
            q = pack_key<FMT>(x[u], d, inv, e, near);
            near = near || !weights_in_range(w_max, e);
            if (((unsure >> u | far >> 8 * u) & 1) || __any_sync(0xffffffffu, near))
                q = exact_key<FMT>(a.qkv + ((size_t)m * n_vec + j) * D, lane, kw, rot, a.eps, d);
        } else if (d == d) {
            q = pack4<FMT>(x[u], d, inv);
        }
        unsigned char* tile = a.pool + ((size_t)page * a.Hkv + h) * kTileBytes;
        uint16_t* dst = reinterpret_cast<uint16_t*>(tile + part * kPartBytes + t * D) + lane;
        dst[0] = (uint16_t)q;
        dst[32] = (uint16_t)(q >> 16);
        if (lane == 0) reinterpret_cast<float*>(tile + kScaleOff)[part * kPageTokens + t] = d;
    }
}

struct Kv8GatherArgs {
    const unsigned char* pool;
    int n_layers, n_pages, Hkv;
    const int* block_table;
    int bt_stride;
    const int* slot;
    const int* t0;           // [M] or nullptr: 0
    const int* n_tok;        // [M]
    const int* row0;         // [M]
    int M, max_tokens, total_rows;
    void* k_out;             // [n_layers][Hkv][total_rows][128]
    void* v_out;
    int* err;
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Gather: one CTA per page of one sequence in one layer; a thread 8 values of one token,
// over the heads' K and V parts, kGatherVecs loads under way at a time. The value d * q is formed
// in f32 and rounded once to the output type.
constexpr int kGatherVecs = 16;                // 8: 1.5 % slower on 32 streams of up to 320 tokens in 28 layers

template <int FMT, typename T>
__global__ void __launch_bounds__(256) kv8_gather_kernel(Kv8GatherArgs a) {
    const int m = blockIdx.y, l = blockIdx.z;
    const int t0 = a.t0 ? a.t0[m] : 0, n = a.n_tok[m], row0 = a.row0[m], slot = a.slot[m];
    if (n == 0) return;
    if (n < 0 || n > a.max_tokens || t0 < 0 || (long long)t0 + n > (long long)a.bt_stride * kPageTokens || row0 < 0 ||
        (long long)row0 + n > a.total_rows || slot < 0) {
        if (blockIdx.x == 0 && l == 0 && threadIdx.x == 0) record_error(a.err, kDevErrBadLen);
        return;
    }
    const int pi = t0 / kPageTokens + blockIdx.x;
    if (pi * kPageTokens >= t0 + n) return;
    const int page = a.block_table[(size_t)slot * a.bt_stride + pi];
    if (page < 0 || page >= a.n_pages) {
        if (threadIdx.x == 0) record_error(a.err, kDevErrBadPage);
        return;
    }
    const int t = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int token = pi * kPageTokens + t;
    if (token < t0 || token >= t0 + n) return;
    const unsigned char* tiles = a.pool + ((size_t)l * a.n_pages + page) * a.Hkv * kTileBytes;
    const size_t row = (size_t)row0 + (token - t0);
    for (int j0 = 0; j0 < 2 * a.Hkv; j0 += kGatherVecs) {
        uint2 w[kGatherVecs];
        float d[kGatherVecs];
#pragma unroll
        for (int u = 0; u < kGatherVecs; ++u) {
            const int j = min(j0 + u, 2 * a.Hkv - 1);
            const unsigned char* tile = tiles + (size_t)(j >> 1) * kTileBytes;
            w[u] = *reinterpret_cast<const uint2*>(tile + (j & 1) * kPartBytes + t * D + 8 * c);
            d[u] = reinterpret_cast<const float*>(tile + kScaleOff)[(j & 1) * kPageTokens + t];
        }
#pragma unroll
        for (int u = 0; u < kGatherVecs; ++u) {
            const int j = j0 + u;
            if (j >= 2 * a.Hkv) break;
            __half2 v[4];
            expand4<FMT>(w[u].x, v[0], v[1]);
            expand4<FMT>(w[u].y, v[2], v[3]);
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(v[i]);
                x[2 * i] = f.x * d[u];
                x[2 * i + 1] = f.y * d[u];
            }
            T* out = reinterpret_cast<T*>((j & 1) ? a.v_out : a.k_out);
            store8(out + (((size_t)l * a.Hkv + (j >> 1)) * a.total_rows + row) * D + 8 * c, x);
        }
    }
}

bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return FA_OK;
    return report_op_error(FA_ERR_CUDA, (std::string(what) + ": " + cudaGetErrorString(e)).c_str());
}

// Whether a warp takes several vectors: once the warps of one vector each would fill the GPU
// (148 SMs x 64 warps); below that more warps shorten the call. One / four a warp (us): append, f16,
// 4800 pairs 2.8 / 3.2, 9600 4.1 / 4.1, 19200 6.4 / 5.7, 76800 22.9 / 18.7; kernel (1), 4736 vectors
// 4.2 / 5.3, 9472 5.2 / 5.9, 14208 6.5 / 6.2, 131072 42.2 / 27.0.
bool several_per_warp(long long vectors) { return vectors > 148 * 64; }

template <int FMT, typename T>
void launch_append(const Kv8AppendArgs& a, unsigned per_row, bool four, cudaStream_t s) {
    const unsigned blocks = (unsigned)a.M * per_row;
    if (four) kv8_append_kernel<FMT, T, 4><<<blocks, 256, 0, s>>>(a, per_row);
    else kv8_append_kernel<FMT, T, 1><<<blocks, 256, 0, s>>>(a, per_row);
}

template <int FMT>
void append_by_type(const Kv8AppendArgs& a, int type, unsigned per_row, bool four, cudaStream_t s) {
    if (type == FA_TYPE_F32) launch_append<FMT, float>(a, per_row, four, s);
    else if (type == FA_TYPE_F16) launch_append<FMT, __half>(a, per_row, four, s);
    else launch_append<FMT, __nv_bfloat16>(a, per_row, four, s);
}

template <int V>
void launch_qkv(const Kv8QkvArgs& a, int format, cudaStream_t s) {
    const dim3 grid(a.M, (a.Hq + 2 * a.Hkv + kQkvWarps * V - 1) / (kQkvWarps * V));
    if (format == FA_KV8_INT8) kv8_qkv_kernel<kInt8, V><<<grid, kQkvWarps * 32, 0, s>>>(a);
    else kv8_qkv_kernel<kE4m3, V><<<grid, kQkvWarps * 32, 0, s>>>(a);
}

template <int FMT>
void gather_by_type(const Kv8GatherArgs& a, int type, dim3 grid, cudaStream_t s) {
    if (type == FA_TYPE_F32) kv8_gather_kernel<FMT, float><<<grid, 256, 0, s>>>(a);
    else if (type == FA_TYPE_F16) kv8_gather_kernel<FMT, __half><<<grid, 256, 0, s>>>(a);
    else kv8_gather_kernel<FMT, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
}

bool known_type(int type) { return type == FA_TYPE_F32 || type == FA_TYPE_F16 || type == FA_TYPE_BF16; }
bool known_format(int format) { return format == FA_KV8_INT8 || format == FA_KV8_E4M3; }

}  // namespace
}  // namespace fa

extern "C" FA_API size_t fa_op_kv8_page_bytes(int n_kv_heads) {
    return n_kv_heads > 0 ? (size_t)n_kv_heads * fa::kv8::kTileBytes : 0;
}

extern "C" FA_API int fa_op_kv8_append(const void* k, const void* v, int src_type, int64_t row_stride, int M,
                                       int n_layers, int n_kv_heads, const int* pos, const int* slot, const int* bt,
                                       int bt_stride, int n_pages, int format, void* pool, int* err, void* stream) {
    using namespace fa;
    if (!k || !v || !pos || !slot || !bt || !pool || M <= 0 || n_layers <= 0 || n_kv_heads <= 0 || bt_stride <= 0 ||
        n_pages <= 0)
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_append: null or non-positive argument");
    if (!known_format(format) || !known_type(src_type))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_append: unknown format or source type");
    const int per16 = src_type == FA_TYPE_F32 ? 4 : 8;
    if (row_stride < (int64_t)n_layers * n_kv_heads * kv8::D || row_stride % per16)
        return report_op_error(FA_ERR_INVALID_ARG,
                               "fa_op_kv8_append: row_stride must cover a row and be a multiple of 16 bytes");
    if (misaligned(k, 16) || misaligned(v, 16) || misaligned(pool, 128))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_append: k and v must be 16-byte, pool 128-byte aligned");
    const long long pairs = (long long)n_layers * n_kv_heads;
    if (pairs > 0x7fffffffll)
        return report_op_error(FA_ERR_CAPACITY, "fa_op_kv8_append: too many vectors for one call");
    const bool four = several_per_warp(M * pairs);
    const long long per_row = four ? (pairs + 31) / 32 : (pairs + 7) / 8;
    if (M * per_row > 0x7fffffffll)
        return report_op_error(FA_ERR_CAPACITY, "fa_op_kv8_append: too many vectors for one call");
    Kv8AppendArgs a{k, v, row_stride, M, n_layers, n_kv_heads, pos, slot, bt, bt_stride, n_pages,
                    static_cast<unsigned char*>(pool), err};
    if (format == FA_KV8_INT8) append_by_type<kv8::kInt8>(a, src_type, (unsigned)per_row, four, (cudaStream_t)stream);
    else append_by_type<kv8::kE4m3>(a, src_type, (unsigned)per_row, four, (cudaStream_t)stream);
    return launched("fa_op_kv8_append");
}

extern "C" FA_API int fa_op_qknorm_rope_append_kv8(const float* qkv, int M, int n_heads, int n_kv_heads,
                                                   const int* pos, const int* slot, const int* bt, int bt_stride,
                                                   int n_pages, const float* qn, const float* kn, float eps,
                                                   const float* rope, int max_pos, int format, void* pool_layer,
                                                   float* q_out, int* err, void* stream) {
    using namespace fa;
    if (!qkv || !pos || !slot || !bt || !qn || !kn || !rope || !pool_layer || !q_out || M <= 0 || n_heads <= 0 ||
        n_kv_heads <= 0 || bt_stride <= 0 || n_pages <= 0 || max_pos <= 0)
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_qknorm_rope_append_kv8: null or non-positive argument");
    if (!known_format(format))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_qknorm_rope_append_kv8: unknown format");
    if (misaligned(qkv, 16) || misaligned(q_out, 16) || misaligned(rope, 16) || misaligned(qn, 8) ||
        misaligned(kn, 8) || misaligned(pool_layer, 128))
        return report_op_error(FA_ERR_INVALID_ARG,
                               "fa_op_qknorm_rope_append_kv8: qkv, rope and q_out must be 16-byte, the norm "
                               "weights 8-byte, the pool 128-byte aligned");
    if ((long long)n_heads + 2ll * n_kv_heads > 65535)
        return report_op_error(FA_ERR_CAPACITY, "fa_op_qknorm_rope_append_kv8: too many heads");
    Kv8QkvArgs a{qkv, M, n_heads, n_kv_heads, pos, slot, bt, bt_stride, n_pages, qn, kn, eps,
                 1.0f / std::sqrt((float)kv8::D), reinterpret_cast<const float2*>(rope), max_pos,
                 static_cast<unsigned char*>(pool_layer), q_out, err};
    const long long n_vec = (long long)n_heads + 2ll * n_kv_heads;
    if (several_per_warp(M * n_vec)) launch_qkv<4>(a, format, (cudaStream_t)stream);
    else launch_qkv<1>(a, format, (cudaStream_t)stream);
    return launched("fa_op_qknorm_rope_append_kv8");
}

extern "C" FA_API int fa_op_kv8_gather(const void* pool, int format, int n_layers, int n_pages, int n_kv_heads,
                                       const int* bt, int bt_stride, const int* slot, const int* t0, const int* n_tok,
                                       const int* row0, int M, int max_tokens, int total_rows, int out_type,
                                       void* k_out, void* v_out, int* err, void* stream) {
    using namespace fa;
    if (!pool || !bt || !slot || !n_tok || !row0 || !k_out || !v_out || M <= 0 || n_layers <= 0 || n_pages <= 0 ||
        n_kv_heads <= 0 || bt_stride <= 0 || max_tokens <= 0 || total_rows <= 0)
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_gather: null or non-positive argument");
    if (!known_format(format) || !known_type(out_type))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_gather: unknown format or output type");
    if (M > 65535 || n_layers > 65535)
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_gather: M and n_layers are limited to 65535");
    if (misaligned(k_out, 16) || misaligned(v_out, 16) || misaligned(pool, 128))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_kv8_gather: outputs must be 16-byte, pool 128-byte aligned");
    if ((long long)bt_stride * kPageTokens > (1ll << 30))
        return report_op_error(FA_ERR_CAPACITY, "fa_op_kv8_gather: bt_stride * 16 is limited to 2^30 tokens");
    Kv8GatherArgs a{static_cast<const unsigned char*>(pool), n_layers, n_pages, n_kv_heads, bt, bt_stride, slot, t0,
                    n_tok, row0, M, max_tokens, total_rows, k_out, v_out, err};
    // a range that does not start on a page boundary spans one page more
    const int pages = (int)std::min<long long>((max_tokens + 2ll * (kPageTokens - 1)) / kPageTokens, bt_stride);
    const dim3 grid(pages, M, n_layers);
    if (format == FA_KV8_INT8) gather_by_type<kv8::kInt8>(a, out_type, grid, (cudaStream_t)stream);
    else gather_by_type<kv8::kE4m3>(a, out_type, grid, (cudaStream_t)stream);
    return launched("fa_op_kv8_gather");
}
