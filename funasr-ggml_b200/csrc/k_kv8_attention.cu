// Decode attention over the 8-bit page pool (formulas in k_kv8_attn.cuh).
#include "k_kv8_attn.cuh"

#include <algorithm>
#include <cmath>
#include <string>

namespace fa {

using namespace kv8;

namespace {

bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace

// The arguments that decode and prefill share, checked; FA_OK or the recorded error.
int kv8_attention_check(const char* what, const Kv8AttnArgs& a, int format, const void* scratch,
                        size_t scratch_bytes, size_t need) {
    auto refuse = [&](int code, const std::string& why) { return report_op_error(code, (what + why).c_str()); };
    if (!a.q || !a.pos || !a.slot || !a.block_table || !a.pool || (!a.out16 && !a.out32) || a.M <= 0 || a.Hq <= 0 ||
        a.Hkv <= 0 || a.bt_stride <= 0 || a.n_pages <= 0)
        return refuse(FA_ERR_INVALID_ARG, ": null or non-positive argument");
    if (a.out16_lo && !a.out16)
        return refuse(FA_ERR_INVALID_ARG, ": out16_lo needs out16");
    if (format != FA_KV8_INT8 && format != FA_KV8_E4M3)
        return refuse(FA_ERR_INVALID_ARG, ": unknown format");
    if (a.Hq % a.Hkv || a.Hq / a.Hkv > 8)
        return refuse(FA_ERR_INVALID_ARG, ": n_heads must be 1 to 8 times n_kv_heads");
    if (misaligned(a.q, 16) || misaligned(a.pool, 128) || misaligned(a.out16, 16) || misaligned(a.out16_lo, 16) ||
        misaligned(a.out32, 16) || misaligned(scratch, 16))
        return refuse(FA_ERR_INVALID_ARG, ": q, outputs and scratch must be 16-byte, pool 128-byte aligned");
    if (a.Hq > 65535 || (long long)a.bt_stride * kPageTokens > (1ll << 30))
        return refuse(FA_ERR_CAPACITY, ": n_heads or bt_stride too large");
    if ((long long)a.n_pages * a.Hkv * (kTileBytes / 128) > 0x7fffffffll)
        return refuse(FA_ERR_CAPACITY, ": the pool has too many pages");
    if (need && (!scratch || scratch_bytes < need))
        return refuse(FA_ERR_INVALID_ARG, ": scratch of " + std::to_string(need) + " bytes required");
    return FA_OK;
}

// The pool as rows of 128 bytes (33 a tile: 16 of K, 16 of V, the scales); a box is K and V.
bool make_kv8_tile_map(CUtensorMap* tm, const void* pool, long long rows) {
    return make_map(tm, pool, 64, rows, 64, 2 * kPageTokens, true);
}

namespace {

// ------------------------------------------------------------------ decode --
// The (row, KV head)s, in that order, are one list of units, a unit per page and kItemUnits
// more for the cost of beginning one; every warp of the grid takes ceil(units / warps) of them,
// whatever rows they cover, so all warps stream the same number of pages however ragged the
// rows are. The part of a warp's range in one (row, KV head) is a segment; one that holds all
// of its row's pages writes the output. The others are at most two a warp (its first and its
// last): the CTA joins those of its four warps, and what it shares with other CTAs, again at
// most two partials, goes to scratch un-normalised and is joined by kv8_merge_kernel.
//
// A warp streams its pages through a ring of its own: lane 0 issues one TMA box (32 rows of
// 128 B: K and V of the head in that page, 128 B swizzle, so that the reads below meet no bank
// conflicts) and one bulk copy (their scales) per page. Per page of 16 tokens, on the tensor
// cores with the keys as the 16-row operand (m16n8k16, f16 in, f32 sums):
//   S[16 tokens][8 columns] = K . q     K expanded to f16 exactly; a query head is two columns,
//                                       hi = f16(q') and lo = f16(q' - hi), q' = q scaled by a
//                                       power of two to [1, 2): 22 bits of q
//   softmax: lane (g, t) = (lane / 4, lane % 4) holds tokens g and g + 8 of head t; sums per
//            lane; the running maximum of a head stays until a score exceeds it by kLazy (log2
//            units), which one vote a page finds out
//   O[16 dims x 8][8 columns] += V^T . w   w = p dv as a hi / lo pair, scaled by a power of two
//                                       that takes the page's largest dv to [2^5, 2^6)
// The page's product starts from zero and is added to the running output by one f32 fma per
// value, so the sum over pages is rounded to nearest.
//
// Bound: HBM. 128 rows of 2048 tokens (16 heads on 8, 554 MB of tiles) take 96-99 us: 84 us of
// pages at the rate of a copy, then some 5 us each of start (lengths, split, page look-ups: four
// dependent loads) and of merge; without its arithmetic the kernel takes as long. 12 or 6 warps a
// CTA took 98.6 and 98.9 us, grids of two to four waves 102 to 109, the merge inside the kernel
// (arrival words) 101. Short calls are latency: the loads of the start, and 0.45 us a page and
// warp (K's MMAs, softmax and V's depend on each other). With eight query heads to a KV head long
// batches are bound by issue: 256 rows of 2048 tokens on 4 KV heads 126 us (a copy's rate: 85); 142
// with the maximum exchanged and O rescaled for every page.
constexpr int kWarps = 4;
constexpr int kCtasPerSm = 3;
constexpr int kMaxCtas = 148 * kCtasPerSm;     // one resident wave of a B200
constexpr int kItemUnits = 2;                  // with ranges per warp: 16 ragged rows 25.6 -> 12.8 us

constexpr float kLazy = 8.0f;                  // weights reach 2^(6 + kLazy)
constexpr int kStages = 3;                     // 128 rows x 2048 tokens: 2 stages 93, 3 96, 4 101 us

// Short contexts: a CTA per (row, KV head), whose warps share its pages evenly, needs no list and
// no merge kernel. It is taken while those CTAs are one resident wave and the block table bounds
// the context to so many pages that the uneven rows and idle SMs cost less than they save (us, int8,
// 16 heads on 8, list / CTA per item):
//   1 row of 64 tokens 7.9 / 4.5, 256 8.0 / 6.1, 512 8.9 / 7.8, 1024 9.2 / 11.2
//   16 rows of 256 9.8 / 6.7, 512 11.4 / 8.4, 1024 15.0 / 12.8, 1 to 1024 11.6 / 11.1
//   55 rows of 256 14.2 / 9.2, 1024 29.0 / 24.3, 1 to 1024 21.9 / 20.5, 1 to 2048 31.7 / 34.4
//   128 rows (more than a wave) of 256 23.3 / 24.1, 1024 54.1 / 58.6
// The host sees the table's width alone: short rows of a wide table take the list.
// Up to an item an SM it has eight warps (4 rows of 512: 7.8 us, with four 8.8, with twelve 8.0).
constexpr int kItemWarps = 8;
bool cta_per_item(long long items, int bt_stride) {
    return items <= kMaxCtas && bt_stride <= (items > 64 ? 64 : 32);
}

template <int NT, int W>
struct DecodeSmem {
    unsigned char tiles[W][kStages][2 * kPartBytes];   // K then V, 128 B swizzle
    float scales[W][kStages][2 * kPageTokens];         // K then V
    // the warps' first partials; their last ones go over the warp's ring once it is drained
    float acc[W][4 * NT][D];
    float2 ml[W][2][4 * NT];                               // running maximum (log2 units), sum
    int4 item[W][2];                                       // (row, KV head, first page, pages), row -1: none
    uint64_t bars[W][kStages];
    long long scan[W];
    int np[W][2];
    int start[3];                                               // the CTA's first row, KV head, unit
};

// Scratch: per CTA the place where its units begin, and two partials of every query head.
struct Partials {
    int4* begin;             // [CTAs] (row, KV head, unit, pages of the row), row -1: no work
    float2* ml;              // [CTAs][2][G]
    float* o;                // [CTAs][2][G][128]
    int* chunk;              // [1] units of a CTA
};
__host__ __device__ inline size_t partial_bytes(int G) {
    return (size_t)kMaxCtas * (sizeof(int4) + 2 * G * (sizeof(float2) + D * sizeof(float))) + 16;
}
__host__ __device__ inline Partials partials(void* scratch, int G) {
    Partials p;
    p.o = static_cast<float*>(scratch);
    p.begin = reinterpret_cast<int4*>(p.o + (size_t)kMaxCtas * 2 * G * D);
    p.ml = reinterpret_cast<float2*>(p.begin + kMaxCtas);
    p.chunk = reinterpret_cast<int*>(p.ml + (size_t)kMaxCtas * 2 * G);
    return p;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

__device__ __forceinline__ uint32_t hi_lo(float x) {
    const __half h = __float2half_rn(x);
    const __half l = __float2half_rn(__fsub_rn(x, __half2float(h)));
    return (uint32_t)__half_as_ushort(h) | ((uint32_t)__half_as_ushort(l) << 16);
}

// Stored values of two tokens (words a, b: four dims each) as f16 pairs (a_i, b_i).
template <int FMT>
__device__ __forceinline__ void expand_pairs(uint32_t a, uint32_t b, uint32_t (&v)[4]) {
    if (FMT == kInt8) {
        const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
        const uint32_t lo = __byte_perm(a, b, 0x5140) ^ 0x80808080u, hi = __byte_perm(a, b, 0x7362) ^ 0x80808080u;
        const uint32_t e[4] = {__byte_perm(lo, 0x64646464u, 0x4140), __byte_perm(lo, 0x64646464u, 0x4342),
                               __byte_perm(hi, 0x64646464u, 0x4140), __byte_perm(hi, 0x64646464u, 0x4342)};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = as_u32(__hsub2(*reinterpret_cast<const __half2*>(&e[i]), off));
    } else {
        __half2 x, y;
        expand4<FMT>(__byte_perm(a, b, 0x5140), x, y);
        v[0] = as_u32(x);
        v[1] = as_u32(y);
        expand4<FMT>(__byte_perm(a, b, 0x7362), x, y);
        v[2] = as_u32(x);
        v[3] = as_u32(y);
    }
}

__device__ __forceinline__ int row_pages(const Kv8AttnArgs& a, int m) {
    return row_bad(a, m) ? 0 : (a.pos[m] + kPageTokens) / kPageTokens;
}

// Quotients of non-negative numbers, in 32 bits where they fit (a 64-bit division is a call
// of a few hundred cycles, on every CTA's way to its first load).
__device__ __forceinline__ long long floor_div(long long x, int y) {
    return x >> 32 ? x / y : (long long)((uint32_t)x / (uint32_t)y);
}
__device__ __forceinline__ long long ceil_div(long long x, int y) { return floor_div(x + y - 1, y); }

// A place in the list: unit u of (row m, KV head h), whose first np units are its pages.
struct Place {
    int m, h, u, np;
};
__device__ __forceinline__ void next_item(const Kv8AttnArgs& a, Place& x) {
    x.u = 0;
    if (++x.h < a.Hkv) return;
    x.h = 0;
    do {
        ++x.m;
        x.np = x.m < a.M ? row_pages(a, x.m) : 1;
    } while (x.np == 0);
}
// n units on (past the list's end: m >= M)
__device__ __forceinline__ void skip_units(const Kv8AttnArgs& a, Place& x, int n) {
    while (x.m < a.M && n >= x.np + kItemUnits - x.u) {
        n -= x.np + kItemUnits - x.u;
        next_item(a, x);
    }
    x.u += n;
}
// n pages on; x is a page, and at least n more follow
__device__ __forceinline__ void skip_pages(const Kv8AttnArgs& a, Place& x, int n) {
    while (n >= x.np - x.u) {
        n -= x.np - x.u;
        next_item(a, x);
    }
    x.u += n;
}

// The queries of a KV head: lane (g, t) holds column g = 2 * head + (lo part), dims [32 t,
// 32 t + 32) as the MMA's rows 2t, 2t+1 and 2t+8, 2t+9 in eight steps. Heads from G on: zeros.
__device__ __forceinline__ void load_query(const Kv8AttnArgs& a, const Place& at, int G, int head, int t,
                                           float (&x)[32]) {
    const float4* src = reinterpret_cast<const float4*>(a.q + ((size_t)at.m * a.Hq + at.h * G + head) * D + 32 * t);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float4 v = head < G ? src[k] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        x[4 * k] = v.x;
        x[4 * k + 1] = v.y;
        x[4 * k + 2] = v.z;
        x[4 * k + 3] = v.w;
    }
}
// The f16 pair of a query scaled by a power of two to [1, 2): hi rounds to 11 bits, lo to
// 2^-25 of the largest value; a column keeps one of the two. Returns the factor that takes
// head t's scores to log2 units.
__device__ __forceinline__ float split_query(const float (&x)[32], int g, int t, uint32_t (&b)[8][2]) {
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) amax = fmaxf(amax, fabsf(x[k]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float p2 = pow2_floor(amax), up = pow2_inverse(p2);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const float y0 = x[2 * k] * up, y1 = x[2 * k + 1] * up;
        const __half2 hi = __floats2half2_rn(y0, y1);
        const float2 f = __half22float2(hi);
        const __half2 lo = __floats2half2_rn(__fsub_rn(y0, f.x), __fsub_rn(y1, f.y));
        b[k >> 1][k & 1] = (g & 1) ? as_u32(lo) : as_u32(hi);
    }
    return __shfl_sync(0xffffffffu, p2, 8 * t) * kLog2e;          // held by the lanes of columns 2t, 2t + 1
}

template <int FMT, int NT, int W, bool ITEM>
__global__ void __launch_bounds__(W * 32, W == kWarps ? kCtasPerSm : 1)
    kv8_decode_kernel(const __grid_constant__ CUtensorMap tm_pool, const Kv8AttnArgs a, void* scratch) {
    constexpr int ST = kStages;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    DecodeSmem<NT, W>& S = *reinterpret_cast<DecodeSmem<NT, W>*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    const int G = a.Hq / a.Hkv;
    const Partials part = partials(scratch, G);
    pdl_trigger();

    // the list's length, and where this CTA's chunk begins
    if (tid == 0) {
        tma_prefetch_desc(&tm_pool);
        for (int w = 0; w < W; ++w)
            for (int s = 0; s < ST; ++s) mbar_init(&S.bars[w][s], 1);
        fence_mbar_init();
    }
    // rows without pages: padding is zeroed, one that cannot be served is flagged and left
    auto rows_without_pages = [&] {
        for (int m = blockIdx.x; m < a.M; m += gridDim.x) {
            if (a.pos[m] == -1)
                for (int d = 4 * tid; d < a.Hq * D; d += W * 128)
                    store4(a, (size_t)m * a.Hq * D + d, make_float4(0.0f, 0.0f, 0.0f, 0.0f), 1.0f);
            else if (tid == 0 && row_bad(a, m)) record_error(a.err, kDevErrBadLen);
        }
    };
    Place at{-1, 0, 0, 0};
    int nw = 0;                                  // pages of the warp's range, which begins at `at`
    if (ITEM) {
        at.m = blockIdx.x / a.Hkv;
        at.h = blockIdx.x % a.Hkv;
        at.np = row_pages(a, at.m);
        rows_without_pages();
        __syncthreads();
        if (at.np == 0) return;
        const int per_warp = (at.np + W - 1) / W;
        at.u = min(warp * per_warp, at.np);
        nw = min(per_warp, at.np - at.u);
    } else {
        const int per = (a.M + W * 32 - 1) / (W * 32);
        const int r0 = min(tid * per, a.M), r1 = min(r0 + per, a.M);
        long long mine = 0;
        for (int m = r0; m < r1; ++m) {
            const int np = row_pages(a, m);
            mine += np ? np + kItemUnits : 0;
        }
        long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) S.scan[warp] = incl;
        __syncthreads();
        long long total = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) incl += S.scan[w];
            total += S.scan[w];
        }
        total *= a.Hkv;
        const int per_warp = (int)ceil_div(total, gridDim.x * W);
        const long long begin = (long long)blockIdx.x * W * per_warp;
        const bool work = begin < total;
        long long before = (incl - mine) * a.Hkv;
        if (work && before <= begin && begin < incl * a.Hkv) {
            for (int m = r0; m < r1; ++m) {
                const int np = row_pages(a, m), units = np ? np + kItemUnits : 0;
                if (begin < before + (long long)units * a.Hkv) {
                    const int h = (int)floor_div(begin - before, units);
                    S.start[0] = m;
                    S.start[1] = h;
                    S.start[2] = (int)(begin - before - (long long)h * units);
                    break;
                }
                before += (long long)units * a.Hkv;
            }
        }
        rows_without_pages();
        __syncthreads();
        if (work) {
            at = Place{S.start[0], S.start[1], S.start[2], 0};
            at.np = row_pages(a, at.m);
        }
        if (tid == 0) {
            part.begin[blockIdx.x] = make_int4(at.m, at.h, at.u, at.np);
            if (blockIdx.x == 0) *part.chunk = W * per_warp;
        }
        if (!work) return;

        // the warp's range: per_warp units from `at`
        skip_units(a, at, warp * per_warp);
        {
            Place x = at;
            for (int left = per_warp; left > 0 && x.m < a.M; next_item(a, x)) {
                nw += max(0, min(x.np - x.u, left));
                left -= min(left, x.np + kItemUnits - x.u);
            }
        }
        if (nw > 0 && at.u >= at.np) next_item(a, at);                // begins in the units behind an item's pages
    }
    float qx[NT][32];                            // the first item's queries, under way while its pages are looked up
#pragma unroll
    for (int c = 0; c < NT; ++c) load_query(a, at, nw > 0 ? G : 0, 4 * c + (g >> 1), t, qx[c]);
    // lane l looks up its pages 32 b + l of batch b, a batch ahead
    Place ahead = at;
    if (lane < nw) skip_pages(a, ahead, lane);
    auto look_up = [&](int first, int& row, int& valid) {
        row = 0;
        valid = 0;
        if (first + lane < nw) {
            const int page = a.block_table[(size_t)a.slot[ahead.m] * a.bt_stride + ahead.u];
            if (page >= 0 && page < a.n_pages) {
                row = (page * a.Hkv + ahead.h) * (kTileBytes / 128);
                valid = min(kPageTokens, a.pos[ahead.m] + 1 - ahead.u * kPageTokens);
            } else {
                record_error(a.err, kDevErrBadPage);             // its tokens are left out
            }
            if (first + 32 + lane < nw) skip_pages(a, ahead, 32);
        }
    };
    int row_a, valid_a, row_b, valid_b;
    look_up(0, row_a, valid_a);
    look_up(32, row_b, valid_b);
    auto issue = [&](int i, int row) {           // lane 0
        const int s = i % ST;
        mbar_arrive_expect_tx(&S.bars[warp][s], kTileBytes);
        tma_load_2d(S.tiles[warp][s], &tm_pool, 0, row, &S.bars[warp][s]);
        bulk_copy_g2s(S.scales[warp][s], a.pool + (size_t)row * 128 + kScaleOff, 2 * kPageTokens * sizeof(float),
                      &S.bars[warp][s]);
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) {
        const int row = __shfl_sync(0xffffffffu, row_a, i);
        if (lane == 0 && i < nw) issue(i, row);
    }
    if (lane < 2) S.item[warp][lane] = make_int4(-1, 0, 0, 0);
    __syncwarp();

    bool ok = true;
    int i = 0;                                   // the warp's pages done
    while (i < nw) {
        const int seg = min(at.np - at.u, nw - i);                // pages of this segment
        const int i_end = i + seg, p_begin = at.u;

        uint32_t qb[NT][8][2];
        float qs[NT];                            // score of head t (+ 4): acc * qs in log2 units
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            if (i > 0) load_query(a, at, G, 4 * c + (g >> 1), t, qx[c]);
            qs[c] = split_query(qx[c], g, t, qb[c]);
        }
        float mx[NT], sum[NT], o[NT][16];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            mx[c] = -INFINITY;
            sum[c] = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; ++k) o[c][k] = 0.0f;
        }

        for (; i < i_end && ok; ++i) {
            const int s = i % ST;
            const int valid = __shfl_sync(0xffffffffu, valid_a, i & 31);
            const bool got = mbar_wait_bounded(&S.bars[warp][s], (uint32_t)(i / ST) & 1u);
            if (!__all_sync(0xffffffffu, got)) {
                ok = false;
                break;
            }
            const unsigned char* Kt = S.tiles[warp][s];
            const unsigned char* Vt = Kt + kPartBytes;
            // scores: K rows g and g + 8, dims 32 t .. (16 B chunks 2t, 2t + 1, swizzled by the row)
            float sc[NT][4];
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[c][e] = 0.0f;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int off = ((2 * t + hf) ^ g) * 16;
                const uint4 x = lds128(Kt + g * 128 + off), y = lds128(Kt + (g + 8) * 128 + off);
                const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    __half2 x0, x1, y0, y1;
                    expand4<FMT>(xw[e], x0, x1);
                    expand4<FMT>(yw[e], y0, y1);
                    const uint32_t fa[4] = {as_u32(x0), as_u32(y0), as_u32(x1), as_u32(y1)};
#pragma unroll
                    for (int c = 0; c < NT; ++c) mma16816(sc[c], fa, qb[c][4 * hf + e][0], qb[c][4 * hf + e][1]);
                }
            }
            const float* scale = S.scales[warp][s];
            const float k0 = scale[g], k1 = scale[g + 8];
            const bool in0 = g < valid, in1 = g + 8 < valid;
            const float v0 = in0 ? scale[kPageTokens + g] : 0.0f, v1 = in1 ? scale[kPageTokens + g + 8] : 0.0f;
            // the power of two at the page's largest V scale, over 2^5
            const float back = __uint_as_float(
                max(__reduce_max_sync(0xffffffffu, max(__float_as_uint(v0), __float_as_uint(v1)) & 0x7f800000u),
                    11u << 23) - (5u << 23));
            const float inv = pow2_inverse(back);
            const float u0 = v0 * inv, u1 = v1 * inv;
            float s0[NT], s1[NT];
            bool above = false;
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                s0[c] = in0 ? (sc[c][0] + sc[c][1]) * (k0 * qs[c]) : -INFINITY;
                s1[c] = in1 ? (sc[c][2] + sc[c][3]) * (k1 * qs[c]) : -INFINITY;
                above |= fmaxf(s0[c], s1[c]) - mx[c] > kLazy;   // exact where it decides, which mx + kLazy is not
            }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    float top = fmaxf(s0[c], s1[c]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    top = fmaxf(top, mx[c]);
                    const float alpha = mx[c] == top ? 1.0f : exp2f(mx[c] - top);
                    mx[c] = top;
                    sum[c] *= alpha;
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[c][k] *= alpha;
                }
            }
            uint32_t w0[NT], w1[NT];
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const float p0 = in0 ? ex2(s0[c] - mx[c]) : 0.0f, p1 = in1 ? ex2(s1[c] - mx[c]) : 0.0f;
                sum[c] += p0 + p1;
                w0[c] = hi_lo(in0 ? p0 * u0 : 0.0f);
                w1[c] = hi_lo(in1 ? p1 * u1 : 0.0f);
            }
            // weights as the second operand: column g = 2 * head + (lo part), tokens 2t, 2t+1, 2t+8, 2t+9
            uint32_t wb[NT][2];
            const uint32_t sel = (g & 1) ? 0x7632 : 0x5410;
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const int from = 8 * t + (g >> 1);
                const uint32_t x0 = __shfl_sync(0xffffffffu, w0[c], from);
                const uint32_t y0 = __shfl_sync(0xffffffffu, w0[c], from + 4);
                const uint32_t x1 = __shfl_sync(0xffffffffu, w1[c], from);
                const uint32_t y1 = __shfl_sync(0xffffffffu, w1[c], from + 4);
                wb[c][0] = __byte_perm(x0, y0, sel);
                wb[c][1] = __byte_perm(x1, y1, sel);
            }
            // V rows of those tokens, dims 16 g ..
            uint32_t vw[4][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int tok = 2 * t + (e & 1) + 8 * (e >> 1);
                const uint4 x = lds128(Vt + tok * 128 + ((g ^ (tok & 7)) * 16));
                // bytes behind the last token may be e4m3 NaN, which a zero weight does not cancel
                const bool live = FMT == kInt8 || tok < valid;
                vw[e][0] = live ? x.x : 0u;
                vw[e][1] = live ? x.y : 0u;
                vw[e][2] = live ? x.z : 0u;
                vw[e][3] = live ? x.w : 0u;
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {        // dims 16 g + 4 d ..
                uint32_t lo[4], hi[4];
                expand_pairs<FMT>(vw[0][d], vw[1][d], lo);
                expand_pairs<FMT>(vw[2][d], vw[3][d], hi);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const uint32_t fa[4] = {lo[e], lo[e + 1], hi[e], hi[e + 1]};
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma16816(acc, fa, wb[c][0], wb[c][1]);
                        float& oa = o[c][4 * d + e];
                        float& ob = o[c][4 * d + e + 1];
                        oa = fmaf(acc[0] + acc[1], back, oa);
                        ob = fmaf(acc[2] + acc[3], back, ob);
                    }
                }
            }
            __syncwarp();
            {
                const int k = i + ST;
                const int row = __shfl_sync(0xffffffffu, (k >> 5) == (i >> 5) ? row_a : row_b, k & 31);
                if (lane == 0 && k < nw) {
                    fence_proxy_async_smem();
                    issue(k, row);
                }
            }
            if ((i & 31) == 31) {
                row_a = row_b;
                valid_a = valid_b;
                look_up(i + 33, row_b, valid_b);
            }
        }
        if (!ok) {
            // A wait gave up: flag it, wait (bounded again) for the warp's copies in flight and
            // leave its part out.
            if (lane == 0) record_error(a.err, kDevErrTimeout);
            for (int k = i; k < min(i + ST, nw); ++k) {
                const bool done = mbar_wait_bounded(&S.bars[warp][k % ST], (uint32_t)(k / ST) & 1u);
                (void)__all_sync(0xffffffffu, done);
            }
            i = nw;
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                mx[c] = -INFINITY;
                sum[c] = 0.0f;
#pragma unroll
                for (int k = 0; k < 16; ++k) o[c][k] = 0.0f;
            }
        }
        // lane (g, t): sum of head t, its dims [16 g, 16 g + 16)
        const bool whole = seg == at.np;
        const int which = i_end == seg ? 0 : 1;                   // the warp's first segment, or its last
        float* to = which ? reinterpret_cast<float*>(S.tiles[warp][0]) : &S.acc[warp][0][0];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            float l = sum[c];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int head = 4 * c + t;
            if (whole) {
                if (head < G) store16(a, ((size_t)at.m * a.Hq + at.h * G + head) * D + 16 * g, o[c], l);
            } else {
                if (g == 0) S.ml[warp][which][head] = make_float2(mx[c], l);
                float4* dst = reinterpret_cast<float4*>(to + head * D + 16 * g);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    dst[k] = make_float4(o[c][4 * k], o[c][4 * k + 1], o[c][4 * k + 2], o[c][4 * k + 3]);
            }
        }
        if (!whole && lane == 0) {
            S.item[warp][which] = make_int4(at.m, at.h, p_begin, seg);
            S.np[warp][which] = at.np;
        }
        if (i < nw) next_item(a, at);
    }

    // The warps' partials in list order, lane k the k-th: those of one (row, KV head) are
    // neighbours, a run. Warp w joins the runs of heads w, w + W, ..., lane l dims 4 l ..
    __syncthreads();
    static_assert(2 * W <= 32, "a lane per partial");
    int4 it = make_int4(-1, 0, 0, 0);
    int np = 0;
    if (lane < 2 * W) {
        it = S.item[lane >> 1][lane & 1];
        np = S.np[lane >> 1][lane & 1];
    }
    const uint32_t parts = __ballot_sync(0xffffffffu, it.x >= 0);
    for (int head = warp; head < G; head += W) {
        const float2 ml = it.x >= 0 ? S.ml[lane >> 1][lane & 1][head] : make_float2(-INFINITY, 0.0f);
        for (uint32_t todo = parts; todo;) {
            const int k0 = __ffs(todo) - 1;
            const int m = __shfl_sync(0xffffffffu, it.x, k0), h = __shfl_sync(0xffffffffu, it.y, k0);
            const int p0 = __shfl_sync(0xffffffffu, it.z, k0), pages = __shfl_sync(0xffffffffu, np, k0);
            const bool in_run = it.x == m && it.y == h;
            const uint32_t run = __ballot_sync(0xffffffffu, in_run);
            todo &= ~run;
            const int sum_pages = __reduce_add_sync(0xffffffffu, in_run ? it.w : 0);
            float M = in_run ? ml.x : -INFINITY;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            // a part without a token (maximum -inf) holds zeros; one whose scores are all NaN, NaN
            const float f = ml.x == M ? 1.0f : exp2f(ml.x - M);
            float L = in_run ? ml.y * f : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
            float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (uint32_t r = run; r; r &= r - 1) {
                const int k = __ffs(r) - 1;
                const float* from =
                    (k & 1) ? reinterpret_cast<const float*>(S.tiles[k >> 1][0]) : &S.acc[k >> 1][0][0];
                const float4 v = reinterpret_cast<const float4*>(from + head * D)[lane];
                const float fk = __shfl_sync(0xffffffffu, f, k);
                O.x = fmaf(v.x, fk, O.x);
                O.y = fmaf(v.y, fk, O.y);
                O.z = fmaf(v.z, fk, O.z);
                O.w = fmaf(v.w, fk, O.w);
            }
            if (ITEM || sum_pages == pages) {
                store4(a, ((size_t)m * a.Hq + h * G + head) * D + 4 * lane, O, L);
            } else {
                // the item that the CTA begins inside (or with) goes to its first slot, one that it does not
                // end to its second
                const bool first = p0 > 0 || (m == S.start[0] && h == S.start[1] && S.start[2] == 0);
                const size_t slot = ((size_t)2 * blockIdx.x + (first ? 0 : 1)) * G + head;
                reinterpret_cast<float4*>(part.o + slot * D)[lane] = O;
                if (lane == 0) part.ml[slot] = make_float2(M, L);
            }
        }
    }
}

// Joins the partials of the (row, KV head)s that several CTAs of the decode kernel share: for
// each CTA c that begins among the pages of one, if c is the first to do so. A block looks at
// eight such c and one query head of each: a warp joins up to eight partials alone, and the
// block's warps together those of an item with more.
constexpr int kMergeWarps = 8;

struct MergeItem {
    int4 at;                 // where CTA c begins
    int c, n, first;         // n partials: slot `first`, then slots 2 c, 2 (c + 1), ...
};
__device__ __forceinline__ MergeItem merge_item(const Partials& part, int c, int n_ctas, int chunk) {
    MergeItem x;
    x.c = c;
    x.n = 0;
    if (c >= n_ctas) return x;
    x.at = part.begin[c];
    // units [0, at.z) of the item lie before CTA c; is c the first CTA that begins among its pages?
    if (x.at.x < 0 || x.at.z == 0 || x.at.z > chunk || x.at.z >= x.at.w) return x;
    x.n = 1 + (x.at.w - x.at.z + chunk - 1) / chunk;
    x.first = 2 * (c - 1) + (x.at.z == chunk ? 0 : 1);
    return x;
}

// Partials k0, k0 + step, ... (at most eight) of an item joined to (M, L, O), lane l dims 4 l ..
__device__ __forceinline__ void merge_eight(const Partials& part, const MergeItem& x, int G, int head, int k0, int step,
                                            int lane, float& M, float& L, float4& O) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int k = k0 + j * step;
        ml[j] = make_float2(-INFINITY, 0.0f);
        v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < x.n) {
            const size_t slot = (size_t)(k ? 2 * (x.c + k - 1) : x.first) * G + head;
            ml[j] = part.ml[slot];
            v[j] = reinterpret_cast<const float4*>(part.o + slot * D)[lane];
        }
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, ml[j].x);
    const float f = M == top ? 1.0f : exp2f(M - top);
    M = top;
    L *= f;
    O = make_float4(O.x * f, O.y * f, O.z * f, O.w * f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float fj = ml[j].x == top ? 1.0f : exp2f(ml[j].x - top);
        L = fmaf(ml[j].y, fj, L);
        O.x = fmaf(v[j].x, fj, O.x);
        O.y = fmaf(v[j].y, fj, O.y);
        O.z = fmaf(v[j].z, fj, O.z);
        O.w = fmaf(v[j].w, fj, O.w);
    }
}

__global__ void __launch_bounds__(kMergeWarps * 32) kv8_merge_kernel(const Kv8AttnArgs a, void* scratch, int n_ctas) {
    __shared__ float4 s_o[kMergeWarps][32];
    __shared__ float2 s_ml[kMergeWarps];
    __shared__ MergeItem s_item[kMergeWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hkv, head = blockIdx.y;
    const Partials part = partials(scratch, G);
    pdl_wait();
    const MergeItem mine = merge_item(part, blockIdx.x * kMergeWarps + warp + 1, n_ctas, *part.chunk);
    if (lane == 0) s_item[warp] = mine;
    if (mine.n > 0 && mine.n <= 8) {
        float M = -INFINITY, L = 0.0f;
        float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        merge_eight(part, mine, G, head, 0, 1, lane, M, L, O);
        store4(a, ((size_t)mine.at.x * a.Hq + mine.at.y * G + head) * D + 4 * lane, O, L);
    }
    if (!__syncthreads_or(mine.n > 8)) return;
    for (int j = 0; j < kMergeWarps; ++j) {
        const MergeItem x = s_item[j];
        if (x.n <= 8) continue;
        float M = -INFINITY, L = 0.0f;
        float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = warp; k < x.n; k += 8 * kMergeWarps) merge_eight(part, x, G, head, k, kMergeWarps, lane, M, L, O);
        s_o[warp][lane] = O;
        if (lane == 0) s_ml[warp] = make_float2(M, L);
        __syncthreads();
        if (warp == 0) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kMergeWarps; ++w) top = fmaxf(top, s_ml[w].x);
            L = 0.0f;
            O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kMergeWarps; ++w) {
                const float f = s_ml[w].x == top ? 1.0f : exp2f(s_ml[w].x - top);
                const float4 v = s_o[w][lane];
                L = fmaf(s_ml[w].y, f, L);
                O.x = fmaf(v.x, f, O.x);
                O.y = fmaf(v.y, f, O.y);
                O.z = fmaf(v.z, f, O.z);
                O.w = fmaf(v.w, f, O.w);
            }
            store4(a, ((size_t)x.at.x * a.Hq + x.at.y * G + head) * D + 4 * lane, O, L);
        }
        __syncthreads();
    }
}

template <int FMT, int NT>
cudaError_t launch_decode(const CUtensorMap& tm, const Kv8AttnArgs& a, void* scratch, cudaStream_t s) {
    const long long items = (long long)a.M * a.Hkv;
    const bool per_item = cta_per_item(items, a.bt_stride);
    if (per_item && items <= 148) {
        kv8_decode_kernel<FMT, NT, kItemWarps, true>
            <<<(int)items, kItemWarps * 32, sizeof(DecodeSmem<NT, kItemWarps>), s>>>(tm, a, scratch);
        return cudaGetLastError();
    }
    if (per_item) {
        kv8_decode_kernel<FMT, NT, kWarps, true>
            <<<(int)items, kWarps * 32, sizeof(DecodeSmem<NT, kWarps>), s>>>(tm, a, scratch);
        return cudaGetLastError();
    }
    // no more CTAs than there can be pages (33 at least: fewer are a CTA per item)
    const int grid = (int)std::min<long long>(items * a.bt_stride, kMaxCtas);
    kv8_decode_kernel<FMT, NT, kWarps, false>
        <<<grid, kWarps * 32, sizeof(DecodeSmem<NT, kWarps>), s>>>(tm, a, scratch);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // launched while the decode kernel runs; it waits for that kernel's end before it reads
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((grid - 1 + kMergeWarps - 1) / kMergeWarps, a.Hq / a.Hkv);
    cfg.blockDim = dim3(kMergeWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv8_merge_kernel, a, scratch, grid);
}

template <int FMT, int NT>
void configure_decode() {
    const cudaFuncAttribute attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaFuncSetAttribute(kv8_decode_kernel<FMT, NT, kWarps, false>, attr, (int)sizeof(DecodeSmem<NT, kWarps>));
    cudaFuncSetAttribute(kv8_decode_kernel<FMT, NT, kWarps, true>, attr, (int)sizeof(DecodeSmem<NT, kWarps>));
    cudaFuncSetAttribute(kv8_decode_kernel<FMT, NT, kItemWarps, true>, attr, (int)sizeof(DecodeSmem<NT, kItemWarps>));
}

}  // namespace

// Opt the kernels into their dynamic shared memory on the current device.
void configure_kv8_attention() {
    configure_decode<kInt8, 1>();
    configure_decode<kInt8, 2>();
    configure_decode<kE4m3, 1>();
    configure_decode<kE4m3, 2>();
}

}  // namespace fa

extern "C" FA_API size_t fa_op_attention_kv8_scratch_bytes(int M, int n_heads, int n_kv_heads) {
    if (M <= 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || n_heads % n_kv_heads) return 0;
    return fa::partial_bytes(n_heads / n_kv_heads);
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
    if (int rc = kv8_attention_check("fa_op_paged_attention_kv8", a, format, scratch, scratch_bytes,
                       fa_op_attention_kv8_scratch_bytes(M, n_heads, n_kv_heads)))
        return rc;
    if (int rc = ensure_device_configured()) return report_op_error(rc, "fa_op_paged_attention_kv8: no CUDA device");
    CUtensorMap tm;
    if (!make_kv8_tile_map(&tm, pool_layer, (long long)n_pages * n_kv_heads * (kTileBytes / 128)))
        return report_op_error(FA_ERR_CUDA, "fa_op_paged_attention_kv8: cannot build the page-pool tensor map");
    const bool wide = n_heads / n_kv_heads > 4;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (format == FA_KV8_INT8)
        e = wide ? launch_decode<kInt8, 2>(tm, a, scratch, st) : launch_decode<kInt8, 1>(tm, a, scratch, st);
    else
        e = wide ? launch_decode<kE4m3, 2>(tm, a, scratch, st) : launch_decode<kE4m3, 1>(tm, a, scratch, st);
    if (e == cudaSuccess) return FA_OK;
    cudaGetLastError();
    return report_op_error(FA_ERR_CUDA, (std::string("fa_op_paged_attention_kv8: ") + cudaGetErrorString(e)).c_str());
}
