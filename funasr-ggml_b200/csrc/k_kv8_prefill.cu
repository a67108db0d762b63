// Causal attention of prefill tiles over the 8-bit page pool on the 5th-generation tensor
// cores (formulas in k_kv8_attn.cuh).
//
// A CTA takes one tile (up to R = 128 / G rows of one sequence, G query heads to a KV head), one
// KV head and, where a call has few tiles, a part of the tile's keys: its up to 128 query
// vectors (vector v = row v % R, head v / R) are the M side of every MMA, so a page is read and
// expanded to f16 once for all of them. Per block of 64 keys (4 pages):
//   S  = Q . K^T        tcgen05.mma kind::f16, M 128, N 64, K 128; Q as the pair hi = f16(q'),
//                       lo = f16(q' - hi), q' = q log2(e) / qs, qs the power of two that takes the
//                       largest to [0.72, 1.44): 22 bits
//   p  = exp2(qs (dk S - m))  one query vector per thread; w = p dv / sigma, sigma a power of two
//                       under the largest dv that the row has seen: f16 pairs, written over S in TMEM
//   O += w . V          M 128, N 128 (dims), K 64 (keys), V MN-major
// A pair's rounding is 2^-25 at most, against 4 or more for the largest V at the running maximum:
// an output is off by 2^-27 a key, as they fall together much less, of the largest |V| that its
// row attends to (and of nothing that it does not attend to).
// w and Q's high parts, the A operands of three quarters of the MMAs, are in TMEM: with all of Q
// and w in shared memory a block would read 160 KB of it for its MMAs (1280 cycles at 128 bytes a
// cycle, 768 as it is), against 1024 cycles that they take. The running maximum is lazy: O is
// rescaled when a block exceeds it by 2^kLazy or sigma grows. qs is a power of two so that qs m is
// exact: rounded by itself, the maximum of scores of 1e8 and more would lie several log2 units from
// the scores that it is taken off.
//
// Roles (512 threads): warp 0 issues the page copies (one TMA box and one bulk copy of scales
// per page) into a ring of raw blocks; warps 4-7 expand a raw block into the f16 K / V tiles of
// a second ring, with each key's factors; warp 1 holds TMEM and issues the MMAs; warps 8-11 and
// 12-15 load Q, run the softmax of the even and of the odd blocks and write the outputs. Every
// mbarrier wait is bounded; on a timeout the CTA records the error, drains its copies and MMAs
// and frees TMEM.
//
// Bound: per block of 64 keys and 128 query vectors the MMAs take 1160 cycles (with the pairs'
// second products twice those of plain f16) and the kernel about 1500: the way from S over the
// softmax to O is longer than the MMAs between, and a rescale or a late page on it is not made up
// for. 4 chunks of 417 to 512 rows at 3500 tokens (16 query heads on 8, 248 CTAs of one SM each)
// take 119 us; 300 with one softmax group, 174 with two S buffers, 142 to 155 with masked and
// whole blocks in one pass, 146 with each block halved between the groups (ten rescales a warp,
// each on the way of the next product). A chunk of 112 rows takes 13.5 to 13.8 us; one chunk of 512 rows
// (64 CTAs, two parts each) 43 us at 3500 tokens and 129 at 16000.
// A persistent form with an even split of the blocks took 160 and 26: every change of tile costs
// 10 us of queries, joins and output, which separate CTAs overlap.
#include "k_attn_body.cuh"
#include "k_kv8_attn.cuh"

#include <algorithm>

namespace fa {

using namespace kv8;

namespace {

constexpr int KB = 64;                        // keys per block
constexpr int PAGES = KB / kPageTokens;
constexpr int RAW = 3;                        // raw ring (8-bit blocks)
constexpr int TILES = 4;                      // f16 ring
constexpr int THREADS = 512;
constexpr int kRegsIssue = 32, kRegsExpand = 64, kRegsSoftmax = 208;
static_assert(kRegsIssue + kRegsExpand + 2 * kRegsSoftmax <= 4 * 128, "registers of the launch");
// Blocks summed in TMEM at a time. The tensor core's f32 sums are truncated, so their error grows
// with their length (2.0e-6 of the output over 57 blocks, 1.2e-6 with stretches of 32); stretches
// are joined in f32 arithmetic rounded to nearest, which costs 1 %.
constexpr int STRETCH = 32;
// Key ranges of one tile and head, and blocks of a range at least: more ranges spread a long context
// over more SMs, and each costs a start and a share of the join. 64 rows on 8 KV heads at 16000 / 40000
// keys with up to 8, 16, 32 ranges: 40 / 82, 30 / 52, 29 / 48 us; at 512 / 1024 / 3500 / 16000 keys
// with 4, 8, 16 blocks at least: 16.4 / 16.8 / 19.8 / 30.3, 18.4 / 19.8 / 20.9 / 30.2,
// 18.5 / 25.0 / 28.1 / 30.8 us.
constexpr int kMaxParts = 16;
constexpr int kMinPartBlocks = 8;
// TMEM columns: S / w of block j at 64 (j % 3), O of the even blocks [192, 320) and of the odd
// ones [320, 448), Q hi [448, 512)
constexpr int SBUF = 3;
constexpr uint32_t TMEM_COLS = 512, COL_O = 192, COL_Q = 448;
// A running maximum is set kRoom above the block's and stays until a block exceeds it by kLazy
// (log2 units): weights reach 2^kLazy, and O is rescaled once in kRoom + kLazy. More room rescales
// less and leaves the weights fewer bits (4: as fast, 1.8e-6 of the output instead of 1.2e-6).
constexpr float kLazy = 11.0f, kRoom = 1.0f;
constexpr uint32_t kSigmaShift = 3;           // the largest V scale over sigma is 2^3 to 2^4: w < 2^15

struct PfSmem {
    __half k[TILES][2][KB * 64];              // [dim half][64 tokens][64 dims], 128 B swizzle
    __half v[TILES][2][KB * 64];
    __half q_lo[2][128 * 64];                 // [dim half][128 query vectors][64 dims], swizzled
    unsigned char raw[RAW][PAGES][2 * kPartBytes];
    float raw_scales[RAW][PAGES][2 * kPageTokens];
    float dk[TILES][KB];                      // K scales
    float dv[TILES][KB];                      // V scales / sigma, for rows that see the whole block
    float dv_raw[TILES][KB];                  // V scales, for the others
    float sigma[TILES];                       // of all keys up to the block's last
    int live[128];                            // the query vector has a row that can be served
    float qs[128];                            // the power of two that takes dk S of a query vector to log2 units
    float state[2][3][128];                   // even / odd blocks' maximum, sum and sigma of each vector
    int raw_pages[RAW];                       // bit q: page q of the block was copied
    int pages[TILES];
    uint64_t raw_full[RAW];
    uint64_t raw_empty[RAW];
    uint64_t kv_full[TILES];
    uint64_t kv_empty[TILES];
    uint64_t s_full[SBUF];
    uint64_t p_half[SBUF];                    // weights of the block's first 32 keys are in TMEM
    uint64_t p_ready[SBUF];                   // all of them are
    uint64_t q_ready;
    uint64_t o_done[2];
    uint64_t drain;
    uint32_t tmem_base;
    int pos_last;                             // last key any row of the tile attends to; -1: none
    int slot;
    int err;
    int issued;                               // raw blocks issued, and waited for
    int consumed;
};

// Byte offset of 16-byte chunk `chunk` (0..7) of row `row` in a [rows][128 B] tile with 128 B
// swizzle.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) {
    return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// f16 pair words of (a, b): high parts, and the rest
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2(a, b);
    const float2 f = h2_to_f2(hi);
    lo = pack2(__fsub_rn(a, f.x), __fsub_rn(b, f.y));
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
// tc_mma_f16_ts, tc_mma_f16 and tc_commit by the lane whose `one` is set.
__device__ __forceinline__ void tc_mma_f16_ts_if(uint32_t one, uint32_t tmem_d, uint32_t tmem_a, uint64_t db,
                                                 uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_mma_f16_if(uint32_t one, uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_commit_if(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(one)
        : "memory");
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    return attn::ffma2(a, make_float2(1.0f, 1.0f), b);
}

__device__ __forceinline__ uint2 lds64(const void* p) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(smem_u32(p)));
    return v;
}

// A barrier of warps 8-15.
__device__ __forceinline__ void group_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// The exponent field of x, 0 for an infinity or NaN.
__device__ __forceinline__ uint32_t finite_exponent(float x) {
    const uint32_t e = __float_as_uint(x) & 0x7f800000u;
    return e == 0x7f800000u ? 0u : e;
}

// The key blocks [first, last) of part `part` of an item of nb blocks cut into at most
// max_parts, and the number of parts.
__device__ __forceinline__ int part_blocks(int nb, int max_parts, int part, int& first, int& last) {
    const int parts = max(1, min(max_parts, nb / kMinPartBlocks));
    const int per = (nb + parts - 1) / parts;
    first = min(part * per, nb);
    last = min(first + per, nb);
    return max(1, (nb + per - 1) / max(per, 1));
}

// By one warp: the last key that the rows of a tile attend to (-1: none) and their slot, the
// one of the row that attends furthest.
__device__ __forceinline__ int tile_extent(const Kv8AttnArgs& a, int2 tile, int lane, int& slot) {
    int best = -1, of = 0;
    for (int r = lane; r < tile.y; r += 32) {
        const int m = tile.x + r, pos = a.pos[m], at = a.slot[m];
        if (!row_bad(a, m) && pos > best) {
            best = pos;
            of = at;
        }
    }
    const int last = __reduce_max_sync(0xffffffffu, best);
    of = __shfl_sync(0xffffffffu, of, __ffs(__ballot_sync(0xffffffffu, best == last)) - 1);
    slot = last >= 0 ? of : 0;
    return last;
}
__device__ __forceinline__ bool tile_bad(const Kv8AttnArgs& a, int2 tile) {
    return tile.x < 0 || tile.y < 1 || tile.y > 128 / (a.Hq / a.Hkv) || tile.x > a.M - tile.y;
}

// Un-normalised partials of the parts: o [items][parts][128 vectors][128], ml (maximum in log2
// units, sum) [items][parts][128]; item = tile * Hkv + KV head.
__host__ __device__ inline size_t part_index(const Kv8AttnArgs& a, int tile, int h, int parts, int part) {
    return (((size_t)tile * a.Hkv + h) * parts + part) * 128;
}

// A maximum in log2 units: exact, or NaN (as the outputs are then) where a score passes f32's range.
__device__ __forceinline__ float in_log2(float top, float qs) {
    const float x = __fmul_rn(top, qs);
    return x == INFINITY ? NAN : x;
}

// The second pass over a block's scores (dk S in sv): p = exp2(dk S qs - top2), whose sum is
// returned, and the weights p f (f: V scales over sigma, times `more` where MASKED) as f16 pairs
// to TMEM over S, the first 32 keys' announced at half_bar. Keys not in `seen` weigh nothing: by
// selection, since the maximum may be -inf and a scale NaN.
template <bool MASKED>
__device__ __forceinline__ float2 weights(const uint32_t (&sv)[KB], const float* factors, float more,
                                          const uint32_t (&seen)[2], float qs, float top2, uint32_t ts,
                                          uint64_t* half_bar) {
    const float4* dv = reinterpret_cast<const float4*>(factors);
    const float2 qs2 = make_float2(qs, qs), neg = make_float2(-top2, -top2), minus = make_float2(-1.0f, -1.0f);
    float2 psum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            float4 f = dv[8 * half + (c >> 2)];
            if (MASKED) f = make_float4(f.x * more, f.y * more, f.z * more, f.w * more);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const int i = 32 * half + c + e;
                const float2 x = attn::ffma2(make_float2(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), qs2, neg);
                float2 p = make_float2(ex2(x.x), ex2(x.y));
                float2 w = attn::fmul2(p, e ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
                if (MASKED) {
                    const uint32_t in = seen[half] >> (c + e);
                    p = make_float2(in & 1 ? p.x : 0.0f, in & 2 ? p.y : 0.0f);
                    w = make_float2(in & 1 ? w.x : 0.0f, in & 2 ? w.y : 0.0f);
                }
                psum = add2(psum, p);
                const uint32_t hw = pack2(w.x, w.y);
                const float2 rest = attn::ffma2(h2_to_f2(hw), minus, w);
                hi[(c + e) >> 1] = hw;
                lo[(c + e) >> 1] = pack2(rest.x, rest.y);
            }
        }
        TMEM_ST_X16(ts + 16 * half, hi);
        TMEM_ST_X16(ts + 32 + 16 * half, lo);
        if (half == 0) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(half_bar);
        }
    }
    return psum;
}

template <int FMT>
__global__ void __launch_bounds__(THREADS, 1)
    kv8_prefill_kernel(const __grid_constant__ CUtensorMap tm_pool, const Kv8AttnArgs a, float* part_o,
                       float2* part_ml) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    PfSmem& S = *reinterpret_cast<PfSmem*>(smem_raw);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const int h = blockIdx.x, max_parts = gridDim.z;
    const int G = a.Hq / a.Hkv, R = 128 / G;
    pdl_trigger();

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_pool);
        for (int s = 0; s < RAW; ++s) {
            mbar_init(&S.raw_full[s], 1);
            mbar_init(&S.raw_empty[s], 4);
        }
        for (int s = 0; s < TILES; ++s) {
            mbar_init(&S.kv_full[s], 4);
            mbar_init(&S.kv_empty[s], 1);
        }
        for (int s = 0; s < SBUF; ++s) {
            mbar_init(&S.s_full[s], 1);
            mbar_init(&S.p_ready[s], 128);
            mbar_init(&S.p_half[s], 128);
        }
        mbar_init(&S.o_done[0], 1);
        mbar_init(&S.o_done[1], 1);
        mbar_init(&S.q_ready, 256);
        mbar_init(&S.drain, 1);
        S.err = 0;
        S.issued = 0;
        S.consumed = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem_base)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int2 tile = a.tiles[blockIdx.y];
    const bool bad = tile_bad(a, tile);
    // warps 8-15: 16 query vectors each, lane l dims [4 l, 4 l + 4); vectors without a row are zero
    // (thread t of each four warps looks after vector t later)
    const int my_r = (threadIdx.x & 127) % R, my_head = (threadIdx.x & 127) / R;
    int my_pos = 0, my_slot = 0;
    bool my_bad = false;
    unsigned char* stage = reinterpret_cast<unsigned char*>(S.k[TILES - 1][0]);
    unsigned char* stage2 = reinterpret_cast<unsigned char*>(S.v[TILES - 1][0]);
    if (warp >= 8) {
        float4 qv[16];
        int head = (warp - 8) * 16 / R, r = (warp - 8) * 16 - head * R;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            qv[k] = !bad && head < G && r < tile.y
                        ? reinterpret_cast<const float4*>(a.q + ((size_t)(tile.x + r) * a.Hq + h * G + head) * D)[lane]
                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (++r == R) {
                r = 0;
                ++head;
            }
        }
        if (my_head < G && my_r < tile.y && !bad) {
            my_pos = a.pos[tile.x + my_r];
            my_slot = a.slot[tile.x + my_r];
            my_bad = row_bad(a, tile.x + my_r);
        }
        // Q as a pair: low parts to shared memory as they are, high parts by way of the last tile
        // of the f16 ring, since a lane writes a whole row of TMEM
        const int hf = lane >> 4, chunk = (lane & 15) >> 1;
        const uint32_t sub = (uint32_t)(lane & 1) * 8;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int v = (warp - 8) * 16 + k;
            const float4 x = qv[k];
            const float big = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
            const float p2 = pow2_floor(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big))));
            const float up = 0.5f * kLog2e * pow2_inverse(p2);
            uint2 hi, lo;
            split2(x.x * up, x.y * up, hi.x, lo.x);
            split2(x.z * up, x.w * up, hi.y, lo.y);
            const uint32_t off = sw128(v, chunk) + sub;
            *reinterpret_cast<uint2*>((hf ? stage2 : stage) + off) = hi;
            *reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(S.q_lo[hf]) + off) = lo;
            if (lane == 0) S.qs[v] = 2.0f * p2;
        }
    }
    if (warp == 0) {
        int slot = 0;
        const int pos_last = bad ? -1 : tile_extent(a, tile, lane, slot);
        if (lane == 0) {
            S.pos_last = pos_last;
            S.slot = slot;
        }
    }
    if (bad && threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0) record_error(a.err, kDevErrBadPos);
    // warp 0 goes on to the copies without waiting for the others
    tc_fence_before();
    if (warp == 0) {
        __syncwarp();
        asm volatile("bar.arrive 2, 512;" ::: "memory");
    } else {
        asm volatile("bar.sync 2, 512;" ::: "memory");
    }
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, S.tmem_base, 0);
    const int pos_last = S.pos_last, slot = S.slot;
    int first = 0, last = 0;
    const int parts = part_blocks((pos_last + KB) / KB, max_parts, blockIdx.z, first, last);
    const int n_blocks = bad || blockIdx.z >= parts ? 0 : last - first;

    // 128 registers a thread at launch, of which the softmax warps take over what the others can
    // spare: 128 threads each of kRegsIssue + kRegsExpand + 2 kRegsSoftmax = 4 x 128
    const bool idle = bad || (int)blockIdx.z >= parts;  // nothing issued: on to the TMEM release
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        if (idle) {
        } else if (warp == 0) {
            bool ok = true;
            int ids = 0;                                   // lane l: page 32 b + l of the part
            for (int j = 0; j < n_blocks; ++j) {
                if (j >= RAW)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.raw_empty[j % RAW], (uint32_t)(j / RAW - 1) & 1u));
                if (!ok) break;
                if ((j & 7) == 0) {
                    const int p = (first + j) * PAGES + lane, last_page = pos_last / kPageTokens;
                    ids = p <= last_page ? a.block_table[(size_t)slot * a.bt_stride + p] : -1;
                    if (p <= last_page && (ids < 0 || ids >= a.n_pages)) {
                        ids = -1;                              // its tokens are left out
                        record_error(a.err, kDevErrBadPage);
                    }
                }
                const int s = j % RAW;
                int id[PAGES], have = 0;
#pragma unroll
                for (int q = 0; q < PAGES; ++q) {
                    id[q] = __shfl_sync(0xffffffffu, ids, (j & 7) * PAGES + q);
                    have |= (id[q] >= 0) << q;
                }
                if (lane == 0) {
                    S.raw_pages[s] = have;
                    mbar_arrive_expect_tx(&S.raw_full[s], __popc(have) * kTileBytes);
#pragma unroll
                    for (int q = 0; q < PAGES; ++q) {
                        if (id[q] < 0) continue;
                        const int row = (id[q] * a.Hkv + h) * (kTileBytes / 128);
                        tma_load_2d(S.raw[s][q], &tm_pool, 0, row, &S.raw_full[s]);
                        bulk_copy_g2s(S.raw_scales[s][q], a.pool + (size_t)row * 128 + kScaleOff,
                                      2 * kPageTokens * sizeof(float), &S.raw_full[s]);
                    }
                    S.issued = j + 1;
                }
                __syncwarp();
            }
            if (!ok && lane == 0) S.err = 1;
        } else if (warp == 1) {
            if (n_blocks > 0) {
                // The whole warp runs the loop and one lane issues: the operands of an MMA then stay in
                // uniform registers (issued from a divergent branch, moving them there took longer than
                // the MMAs: 2070 cycles a block).
                constexpr uint32_t kIdS = idesc_f16(128, KB, false, false);
                constexpr uint32_t kIdPV = idesc_f16(128, D, false, true);
                const uint32_t one = elect_one();
                const uint64_t k_desc = smem_desc_k128(S.k[0][0]), v_desc = smem_desc_mn128(S.v[0][0], KB * 64 * 2);
                const uint64_t q_desc = smem_desc_k128(S.q_lo[0]);
                bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.q_ready, 0));
                // S of block j + 2 before O of block j: with three S buffers it needs only block j - 1's
                // product, so a group finds its next S ready when it ends a block
                for (int i = 0; ok && i < n_blocks + 2; ++i) {
                    if (i < n_blocks) {
                        const int s = i % TILES;
                        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.kv_full[s], (uint32_t)(i / TILES) & 1u));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t d_s = tmem + (uint32_t)(i % SBUF * KB);
                        const uint64_t db = k_desc + (uint32_t)(s * (int)sizeof(S.k[0]) >> 4);
                        // the low parts first: the sums are cut off at the size of the low products then, and
                        // only the eight steps of the high parts at that of a score
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk) {
                            const uint64_t in_tile = (kk >> 2) * (int)sizeof(S.k[0][0]) / 16 + (kk & 3) * 32 / 16;
                            const uint64_t in_q = (kk >> 2) * (int)sizeof(S.q_lo[0]) / 16 + (kk & 3) * 32 / 16;
                            tc_mma_f16_if(one, d_s, q_desc + in_q, db + in_tile, kIdS, kk > 0 ? 1u : 0u);
                        }
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk) {
                            const uint64_t in_tile = (kk >> 2) * (int)sizeof(S.k[0][0]) / 16 + (kk & 3) * 32 / 16;
                            tc_mma_f16_ts_if(one, d_s, tmem + COL_Q + 8 * kk, db + in_tile, kIdS, 1u);
                        }
                        tc_commit_if(one, &S.s_full[i % SBUF]);
                    }
                    if (i >= 2) {
                        const int j = i - 2, s = j % TILES;
                        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.p_half[j % SBUF], (uint32_t)(j / SBUF) & 1u));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t d_p = tmem + (uint32_t)(j % SBUF * KB);
                        const uint32_t d_o = tmem + COL_O + (uint32_t)((j & 1) * D);
                        const uint64_t db = v_desc + (uint32_t)(s * (int)sizeof(S.v[0]) >> 4);
                        // the first 32 keys' products as soon as their weights are there
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            if (kk == 2) {
                                ok = __all_sync(0xffffffffu,
                                                mbar_wait_bounded(&S.p_ready[j % SBUF], (uint32_t)(j / SBUF) & 1u));
                                tc_fence_after();
                            }
                            const uint64_t at = db + kk * 16 * 64 * 2 / 16;
                            tc_mma_f16_ts_if(one, d_o, d_p + 8 * kk, at, kIdPV, (j % STRETCH > 1 || kk > 0) ? 1u : 0u);
                            tc_mma_f16_ts_if(one, d_o, d_p + 32 + 8 * kk, at, kIdPV, 1u);
                        }
                        if (!ok) break;
                        tc_commit_if(one, &S.kv_empty[s]);
                        tc_commit_if(one, &S.o_done[j & 1]);
                    }
                }
                tc_commit_if(one, &S.drain);
                if (!mbar_wait_bounded(&S.drain, 0)) ok = false;
                if (!ok && lane == 0) S.err = 1;
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsExpand));
        // expansion: a thread takes 8 bytes, dims 8 c .., of every eighth token, K and V (one 16-byte
        // chunk of the f16 tile each: eight lanes read and write whole rows, without bank conflicts)
        const int ct = threadIdx.x - 128, cw = warp - 4;
        const int c = ct & 15, r = ct >> 4;
        const uint32_t raw_at = r * 128 + (((c >> 1) ^ r) << 4) + (c & 1) * 8;
        uint32_t run = 0;                              // exponent field of sigma
        bool ok = true;
        for (int j = 0; j < n_blocks; ++j) {
            const int s = j % RAW, d = j % TILES;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.raw_full[s], (uint32_t)(j / RAW) & 1u));
            if (ok && j >= TILES)
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.kv_empty[d], (uint32_t)(j / TILES - 1) & 1u));
            if (ok && j == TILES - 1)                  // Q's high parts pass through the last tile (below)
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&S.q_ready, 0));
            if (!ok) break;
            if (ct == 0) S.consumed = j + 1;
            const int have = S.raw_pages[s];
            const int key0 = (first + j) * KB;
            // the keys' factors: sigma covers the finite V scales of the block's tokens
            float dv[2];
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = lane + 32 * e;
                const bool in = ((have >> (t >> 4)) & 1) && key0 + t <= pos_last;
                dv[e] = in ? S.raw_scales[s][t >> 4][kPageTokens + (t & 15)] : 0.0f;
                top = max(top, finite_exponent(dv[e]));
            }
            top = max(__reduce_max_sync(0xffffffffu, top), 11u << 23);
            run = max(run, top);
            if (cw == 0) {
                const float sigma = __uint_as_float(run - (kSigmaShift << 23)), inv = pow2_inverse(sigma);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int t = lane + 32 * e;
                    S.dk[d][t] = S.raw_scales[s][t >> 4][t & 15];
                    S.dv[d][t] = dv[e] * inv;
                    S.dv_raw[d][t] = dv[e];
                }
                if (lane == 0) {
                    S.sigma[d] = sigma;
                    S.pages[d] = have;
                }
            }
            // token 8 i + r of the block, dims 8 c ..: all loads of K (then V) before the first store
            unsigned char* k_out = reinterpret_cast<unsigned char*>(S.k[d][c >> 3]) + sw128(r, c & 7);
            unsigned char* v_out = reinterpret_cast<unsigned char*>(S.v[d][c >> 3]) + sw128(r, c & 7);
            const bool whole = have == (1 << PAGES) - 1 && key0 + KB - 1 <= pos_last;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                uint2 x[KB / 8];
#pragma unroll
                for (int i = 0; i < KB / 8; ++i)
                    x[i] = lds64(S.raw[s][i >> 1] + part * kPartBytes + (i & 1) * 1024 + raw_at);
                // tokens of pages left out, and V behind the last token (unwritten bytes may be e4m3 NaN)
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < KB / 8; ++i)
                        if (!((have >> (i >> 1)) & 1) || (part && key0 + 8 * i + r > pos_last)) x[i] = make_uint2(0, 0);
                }
#pragma unroll
                for (int i = 0; i < KB / 8; ++i) {
                    __half2 y[4];
                    expand4<FMT>(x[i].x, y[0], y[1]);
                    expand4<FMT>(x[i].y, y[2], y[3]);
                    *reinterpret_cast<uint4*>((part ? v_out : k_out) + i * 1024) = *reinterpret_cast<const uint4*>(y);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&S.kv_full[d]);
                mbar_arrive(&S.raw_empty[s]);
            }
        }
        if (!ok && lane == 0) S.err = 1;
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        if (!idle) {
            // Warps 8-11 the even blocks, 12-15 the odd ones, each with its own running maximum, sum
            // and O: while one group works on S of a block, the MMAs make the other's. Thread t of a
            // group owns TMEM lane t = query vector t (a warp may only touch lanes 32 * (warp % 4) ..).
            const int odd = warp >= 12 ? 1 : 0;
            const int quarter = warp & 3;
            const int t = 32 * quarter + lane;
            bool live = my_head < G && my_r < tile.y;
            int pos = pos_last;                        // lanes without a row mask no more than the others
            if (live) {
                pos = my_pos;
                if (my_bad || (pos >= 0 && my_slot != slot)) {
                    if (h == 0 && blockIdx.z == 0 && my_head == 0 && !odd) record_error(a.err, kDevErrBadLen);
                    live = false;
                    pos = pos_last;
                }
            }
            const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16);
            if (n_blocks > 0) {
                // each group writes half of the dims
                uint32_t row_hi[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 x = lds128((odd ? stage2 : stage) + sw128(t, c));
                    row_hi[4 * c] = x.x;
                    row_hi[4 * c + 1] = x.y;
                    row_hi[4 * c + 2] = x.z;
                    row_hi[4 * c + 3] = x.w;
                }
                TMEM_ST_X32(tl + COL_Q + 32 * odd, row_hi);
                tmem_wait_st();
                fence_proxy_async_smem();
                tc_fence_before();
                mbar_arrive(&S.q_ready);
            }
            const float qs = n_blocks > 0 ? S.qs[t] : 0.0f;
            const float lazy = fminf(kLazy / qs, 1e37f), room = fminf(kRoom / qs, 1e37f);
            const uint32_t to = tl + COL_O + (uint32_t)(odd * D);
            const size_t at = part_index(a, blockIdx.y, h, max_parts, blockIdx.z) + t;
            // over the stretches joined so far: maximum, sum, and the group's half of the dims
            float all_max = -INFINITY, all_sum = 0.0f, acc[64];
#pragma unroll
            for (int e = 0; e < 64; ++e) acc[e] = 0.0f;
            bool ok = true;
            // running maximum of dk S (before qs), the same in log2 units, and sigma
            float top = -INFINITY, top2 = -INFINITY, sigma = 0.0f;
            for (int j0 = 0; j0 == 0 || j0 < n_blocks; j0 += STRETCH) {
                const int j1 = min(j0 + STRETCH, n_blocks);
                float sum = 0.0f;                      // of the stretch's weights
                for (int j = j0 + odd; ok && j < j1; j += 2) {
                    const int d = j % TILES;
                    const bool got = mbar_wait_bounded(&S.kv_full[d], (uint32_t)(j / TILES) & 1u) &&
                                     mbar_wait_bounded(&S.s_full[j % SBUF], (uint32_t)(j / SBUF) & 1u);
                    if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t ts = tl + (uint32_t)(j % SBUF * KB);
                    uint32_t sv[KB];
                    TMEM_LD_X32(ts, sv);
                    TMEM_LD_X32(ts + 32, (sv + 32));
                    tmem_wait_ld();
                    const int key0 = (first + j) * KB;
                    const int have = S.pages[d];
                    const bool masked = !__all_sync(0xffffffffu, key0 + KB - 1 <= pos && have == (1 << PAGES) - 1);
                    const float4* dk = reinterpret_cast<const float4*>(S.dk[d]);
                    float bmax = -INFINITY;
#pragma unroll
                    for (int c = 0; c < KB; c += 4) {
                        const float4 f = dk[c >> 2];
                        const float2 x = attn::fmul2(make_float2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])),
                                                     make_float2(f.x, f.y));
                        const float2 y =
                            attn::fmul2(make_float2(__uint_as_float(sv[c + 2]), __uint_as_float(sv[c + 3])),
                                        make_float2(f.z, f.w));
                        sv[c] = __float_as_uint(x.x);
                        sv[c + 1] = __float_as_uint(x.y);
                        sv[c + 2] = __float_as_uint(y.x);
                        sv[c + 3] = __float_as_uint(y.y);
                    }
                    uint32_t seen[2] = {~0u, ~0u};             // keys of the block that the row attends to
                    if (masked) {
                        const int n = min(max(pos + 1 - key0, 0), KB);
                        uint64_t bits = n == KB ? ~0ull : (1ull << n) - 1;
#pragma unroll
                        for (int q = 0; q < PAGES; ++q)
                            if (!((have >> q) & 1)) bits &= ~(0xffffull << (16 * q));
                        seen[0] = (uint32_t)bits;
                        seen[1] = (uint32_t)(bits >> 32);
#pragma unroll
                        for (int c = 0; c < KB; ++c)
                            if (!((seen[c >> 5] >> (c & 31)) & 1)) sv[c] = 0xff800000u;        // -inf
                    }
#pragma unroll
                    for (int c = 0; c < KB; ++c) bmax = fmaxf(bmax, __uint_as_float(sv[c]));
                    // a sigma of the row's own where it does not see every key: a large V that it may not see must
                    // not scale its weights away
                    float next_sigma = S.sigma[d];
                    if (masked) {
                        const float4* raw = reinterpret_cast<const float4*>(S.dv_raw[d]);
                        uint32_t own = 11u << 23;
#pragma unroll
                        for (int c = 0; c < KB; c += 4) {
                            const float4 f = raw[c >> 2];
                            const uint32_t in = seen[c >> 5] >> (c & 31);
                            if (in & 1) own = max(own, finite_exponent(f.x));
                            if (in & 2) own = max(own, finite_exponent(f.y));
                            if (in & 4) own = max(own, finite_exponent(f.z));
                            if (in & 8) own = max(own, finite_exponent(f.w));
                        }
                        next_sigma = fmaxf(sigma, __uint_as_float(own - (kSigmaShift << 23)));
                    }
                    float alpha = j - j0 > 1 ? sigma * pow2_inverse(next_sigma) : 1.0f;
                    sigma = next_sigma;
                    if (top == -INFINITY) {
                        top = bmax + room;                     // first block with a key: O holds nothing of this row
                        top2 = in_log2(top, qs);
                    } else if (bmax - top > lazy) {            // exact where it decides, which top + lazy is not
                        top = bmax + room;
                        const float next = in_log2(top, qs);
                        const float f = exp2f(top2 - next);
                        top2 = next;
                        alpha *= f;
                        sum *= f;
                    }
                    if (j - j0 > 1 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                        const bool od = mbar_wait_bounded(&S.o_done[odd], (uint32_t)((j >> 1) - 1) & 1u);
                        if (!__all_sync(0xffffffffu, od)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t ov[32];
                            TMEM_LD_X32(to + c, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                            TMEM_ST_X32(to + c, ov);
                        }
                    }
                    uint64_t* half_bar = &S.p_half[j % SBUF];
                    const float2 psum =
                        masked ? weights<true>(sv, S.dv_raw[d], pow2_inverse(sigma), seen, qs, top2, ts, half_bar)
                               : weights<false>(sv, S.dv[d], 1.0f, seen, qs, top2, ts, half_bar);
                    sum += psum.x + psum.y;
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&S.p_ready[j % SBUF]);
                }
                // the group's last product of the stretch: block j1 - 1 or j1 - 2
                const int last_j = ((j1 - 1 - odd) & ~1) + odd;
                if (ok && last_j >= j0 && j1 > odd) {
                    const bool od = mbar_wait_bounded(&S.o_done[odd], (uint32_t)(last_j >> 1) & 1u);
                    ok = __all_sync(0xffffffffu, od);
                }
                if (!ok && lane == 0) S.err = 1;
                S.state[odd][0][t] = top2;
                S.state[odd][1][t] = sum;
                S.state[odd][2][t] = sigma;
                tc_fence_before();
                group_sync();
                tc_fence_after();
                if (!S.err) {
                    // the two groups and the stretches before joined: acc = O0 f0 + O1 f1 + fa acc, each group half
                    // of the dims
                    const float m0 = S.state[0][0][t], m1 = S.state[1][0][t], best = fmaxf(fmaxf(m0, m1), all_max);
                    float f0 = m0 == best ? 1.0f : exp2f(m0 - best), f1 = m1 == best ? 1.0f : exp2f(m1 - best);
                    const float fa = all_max == best ? 1.0f : exp2f(all_max - best);
                    all_sum = S.state[0][1][t] * f0 + S.state[1][1][t] * f1 + all_sum * fa;
                    all_max = best;
                    f0 *= S.state[0][2][t];
                    f1 *= S.state[1][2][t];
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        uint32_t ov[16];
                        if (j1 > j0) {
                            TMEM_LD_X16(tl + COL_O + 64 * odd + c, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(__uint_as_float(ov[e]), f0, acc[c + e] * fa);
                        }
                        if (j1 - j0 > 1) {
                            TMEM_LD_X16(tl + COL_O + D + 64 * odd + c, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(__uint_as_float(ov[e]), f1, acc[c + e]);
                        }
                    }
                }
                tc_fence_before();
                group_sync();                                  // O and the state may be written again
                tc_fence_after();
            }
            // the part's un-normalised sum, or the output, by way of the K tiles (no MMA reads them any
            // more), so that a warp stores whole rows: from a row per thread, 112 rows took 3 us longer
            unsigned char* stage = reinterpret_cast<unsigned char*>(S.k[0][0]);
            const float inv = parts > 1 ? 1.0f : all_sum == 0.0f ? 0.0f : 1.0f / all_sum;
            if (parts > 1 && !odd && !S.err) part_ml[at] = make_float2(all_max, all_sum);
            if (!odd) S.live[t] = live;
#pragma unroll
            for (int c = 0; c < 64; c += 4)
                *reinterpret_cast<float4*>(stage + t * 512 + (((16 * odd + (c >> 2)) ^ (t & 7)) << 4)) =
                    make_float4(acc[c] * inv, acc[c + 1] * inv, acc[c + 2] * inv, acc[c + 3] * inv);
            group_sync();
            if (!S.err) {
                const int v0 = (warp - 8) * 16;
                const uint32_t lives = __ballot_sync(0xffffffffu, S.live[v0 + (lane & 15)] != 0);
                float4* to_part = reinterpret_cast<float4*>(part_o + (at - t + v0) * D) + lane;
                int vh = v0 / R, vr = v0 - vh * R;
#pragma unroll 1
                for (int k0 = 0; k0 < 16; k0 += 8) {
                    float4 o[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        o[k] = *reinterpret_cast<const float4*>(stage + (v0 + k0 + k) * 512 + ((lane ^ k) << 4));
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (parts > 1) {
                            to_part[(k0 + k) * (D / 4)] = o[k];
                        } else if ((lives >> (k0 + k)) & 1) {
                            const float x[4] = {o[k].x, o[k].y, o[k].z, o[k].w};
                            store_values<4>(a, ((size_t)(tile.x + vr) * a.Hq + h * G + vh) * D + 4 * lane, x);
                        }
                        if (++vr == R) {
                            vr = 0;
                            ++vh;
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (S.err) {
        if (threadIdx.x == 0) {
            record_error(a.err, kDevErrTimeout);
            for (int j = S.consumed; j < S.issued; ++j)
                (void)mbar_wait_bounded(&S.raw_full[j % RAW], (uint32_t)(j / RAW) & 1u);
        }
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Joins the parts of a tile and KV head: a warp per query vector, lane l dims [4 l, 4 l + 4).
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(const Kv8AttnArgs a, const float* part_o,
                                                               const float2* part_ml, int max_parts) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.Hkv, ti = blockIdx.x / a.Hkv;
    const int G = a.Hq / a.Hkv, R = 128 / G;
    const int2 tile = a.tiles[ti];
    pdl_wait();
    if (tile_bad(a, tile)) return;
    int slot, first, last;
    const int pos_last = tile_extent(a, tile, lane, slot);
    const int parts = part_blocks((pos_last + KB) / KB, max_parts, 0, first, last);
    if (parts == 1) return;
    const int t = blockIdx.y * 8 + warp;
    const int r = t % R, head = t / R, row = tile.x + r;
    if (head >= G || r >= tile.y || row_bad(a, row) || (a.pos[row] >= 0 && a.slot[row] != slot)) return;
    float2 ml[kMaxParts];
    float M = -INFINITY, L = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < kMaxParts; ++k) {
        ml[k] = k < parts ? part_ml[part_index(a, ti, h, max_parts, k) + t] : make_float2(-INFINITY, 0.0f);
        M = fmaxf(M, ml[k].x);
    }
#pragma unroll
    for (int k = 0; k < kMaxParts; ++k) {
        if (k >= parts) break;
        const float4 v = reinterpret_cast<const float4*>(part_o + (part_index(a, ti, h, max_parts, k) + t) * D)[lane];
        // a part without a key (maximum -inf) holds zeros; one whose scores are all NaN, NaN
        const float f = ml[k].x == M ? 1.0f : exp2f(ml[k].x - M);
        L = fmaf(ml[k].y, f, L);
        O.x = fmaf(v.x, f, O.x);
        O.y = fmaf(v.y, f, O.y);
        O.z = fmaf(v.z, f, O.z);
        O.w = fmaf(v.w, f, O.w);
    }
    store4(a, ((size_t)row * a.Hq + h * G + head) * D + 4 * lane, O, L);
}

// Parts that a tile's keys may be cut into: as many as leave the tiles and heads of a call in
// one wave of a B200's 148 SMs (a CTA fills an SM).
int max_parts(int n_tiles, int n_kv_heads) {
    const long long items = (long long)n_tiles * n_kv_heads;
    return (int)std::max<long long>(1, std::min<long long>(kMaxParts, 148 / items));
}

template <int FMT>
cudaError_t launch_prefill(const CUtensorMap& tm, const Kv8AttnArgs& a, void* scratch, cudaStream_t s) {
    const int parts = max_parts(a.n_tiles, a.Hkv);
    float* part_o = static_cast<float*>(scratch);
    float2* part_ml =
        parts > 1 ? reinterpret_cast<float2*>(part_o + (size_t)a.n_tiles * a.Hkv * parts * 128 * D) : nullptr;
    kv8_prefill_kernel<FMT><<<dim3(a.Hkv, a.n_tiles, parts), THREADS, sizeof(PfSmem), s>>>(tm, a, part_o, part_ml);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || parts == 1) return e;
    // launched while the kernel above runs; it waits for that kernel's end before it reads
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_tiles * a.Hkv, 16);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv8_prefill_merge_kernel, a, (const float*)part_o, (const float2*)part_ml, parts);
}

}  // namespace

// Opt the kernels into their dynamic shared memory on the current device.
void configure_kv8_prefill() {
    const cudaFuncAttribute attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaFuncSetAttribute(kv8_prefill_kernel<kInt8>, attr, (int)sizeof(PfSmem));
    cudaFuncSetAttribute(kv8_prefill_kernel<kE4m3>, attr, (int)sizeof(PfSmem));
}

}  // namespace fa

extern "C" FA_API size_t fa_op_prefill_attention_kv8_scratch_bytes(int n_tiles, int n_heads, int n_kv_heads) {
    if (n_tiles <= 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || n_heads % n_kv_heads) return 0;
    const int parts = fa::max_parts(n_tiles, n_kv_heads);
    return parts == 1 ? 0 : (size_t)n_tiles * n_kv_heads * parts * 128 * (fa::D * sizeof(float) + sizeof(float2));
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
    if (!tiles || n_tiles <= 0 || (reinterpret_cast<uintptr_t>(tiles) & 7))
        return report_op_error(FA_ERR_INVALID_ARG, "fa_op_prefill_attention_kv8: tiles missing or not 8-byte aligned");
    if (int rc = kv8_attention_check("fa_op_prefill_attention_kv8", a, format, scratch, scratch_bytes,
                                     fa_op_prefill_attention_kv8_scratch_bytes(n_tiles, n_heads, n_kv_heads)))
        return rc;
    if (n_tiles > 65535)
        return report_op_error(FA_ERR_CAPACITY, "fa_op_prefill_attention_kv8: more than 65535 tiles");
    if (int rc = ensure_device_configured()) return report_op_error(rc, "fa_op_prefill_attention_kv8: no CUDA device");
    CUtensorMap tm;
    if (!make_kv8_tile_map(&tm, pool_layer, (long long)n_pages * n_kv_heads * (kTileBytes / 128)))
        return report_op_error(FA_ERR_CUDA, "fa_op_prefill_attention_kv8: cannot build the page-pool tensor map");
    const cudaError_t e = format == FA_KV8_INT8 ? launch_prefill<kInt8>(tm, a, scratch, (cudaStream_t)stream)
                                                : launch_prefill<kE4m3>(tm, a, scratch, (cudaStream_t)stream);
    if (e == cudaSuccess) return FA_OK;
    cudaGetLastError();
    return report_op_error(FA_ERR_CUDA, (std::string("fa_op_prefill_attention_kv8: ") + cudaGetErrorString(e)).c_str());
}
