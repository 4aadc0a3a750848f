// Attention of many rows (query tokens x heads of a kv head) over the 4-bit
// cache with 16-bit outputs: prompt chunks, on the fifth-generation tensor
// cores.
//
// A CTA takes 256 rows of one kv head as two tiles of 128 and goes through a
// split of the tokens 128 at a time. Its warps have roles, as in the 8-bit
// cache's chunk kernel:
//
//   warps 0-3, 4-7  softmax of tile 0 and 1, one thread per row
//   warps 8-11      K and V: codes from global memory to values in shared
//                   memory (the conversion is shared by all 256 rows)
//   warp 12         one thread issues tcgen05.mma
//
// Thirteen warps leave a thread 128 registers; with four code warps each for K
// and V, and 96 registers, 2048 query tokens of 32768 take 971 us, so 957. Up to
// 128 rows are one tile twice (SHARED), which take every other step: steps come
// faster, and four code warps each for K and V are better, 41 against 45 us
// (8 x 5 tokens, 64/8 heads, to 8192).
//
// S = Q K^T (M 128 rows, N 128 tokens) and O += P V (N head_dim) accumulate in
// tensor memory: two S tiles and two O tiles fill its 512 columns. P is
// written as fp16 over its own S, 64 tokens at a time, and is the A operand of
// the second product. While one tile's softmax runs, the other tile's products
// do. The order of the issues is the order of execution, so an S that is there
// tells that the P V before it is done.
//
// Shared memory operands are K-major with the 128-byte swizzle: Q and K
// [row][d], V transposed to [d][token]. K and V are code * scale, the fp16
// numbers that the format defines: scores and the values' sum need no scale,
// and the softmax no more than one multiplication and addition a score.
//
// Softmax: t = s * factor - base, p = 2^t. `base` follows the row maximum
// loosely: the first tokens set it so that their largest p is 2^6, and only a
// row whose p of 64 tokens add up to more than 2^15 (no p leaves fp16 before)
// moves it and scales O, which after the first tokens hardly ever happens.
// So no maximum is taken. Where a row does not see all of 64 tokens, and where scores
// are so large that fp32 has no bits for differences to the base, S is
// rewritten as t first, -inf for what is not seen.
//
// P is rounded to fp16 (2^-11 of itself at most), and O is added up by the
// tensor cores, which truncate: 6e-9 of it per token of the split.
//
// With head_dim above 128 a CTA has one tile of rows, one stage of K and V, and
// K is warps 4-7, V 8-11, the issuing warp 12 (2 x 512 tokens of 8192, 8/1
// heads, head_dim 256: 108 us; with four code warps for both 132).
//
// Measured, 2048 query tokens of 32768, 32/8 heads, head_dim 128, bf16: 949 us
// in short runs, 1122 TFLOP/s or 67 % of a library product's; 1116 us (954
// TFLOP/s, 68 % of what such products sustain) at the power cap. Of a step of two tiles the
// tensor cores work 60 % of the time, instructions issue in 43 % of the cycles;
// what bounds it is the round S -> softmax -> P -> S of a tile, whose softmax is
// bound by exp2 and the conversions to fp16 (a step's 32768 scores). Two softmax
// warpgroups a tile, half of the columns each, took 1302 us, two issuing warps 1115
// where one took 1010. Short cases are bound by the start: 1 x 512 tokens of 4096 58 us, 39 of
// 75 15 us, of which queries into shared memory 4 and rows out 4.
#pragma once
#include "akv_q4_loads.cuh"
#include "akv_q8_chunk.cuh"

namespace akv {
namespace q4 {

using q8::kChunkHalf;
using q8::kChunkTiles;
using q8::kChunkTokens;
using q8::add2;
using q8::bar_arrive;
using q8::bar_init;
using q8::elect_lane;
using q8::exp2_fast;
using q8::fence_after;
using q8::fence_async;
using q8::fence_before;
using q8::fma2;
using q8::halves;
using q8::mma_commit;
using q8::mma_desc;
using q8::mma_ss;
using q8::mma_ts;
using q8::operand_desc;
using q8::pack_half2;
using q8::pair_of;
using q8::smem_addr;
using q8::swizzled;
using q8::tmem_ld16;
using q8::tmem_st16;
using q8::tmem_wait_ld;
using q8::tmem_wait_st;

// Tries of a wait: one takes about 4.5 us, all some 19 s.
constexpr int kWaitTries = 1 << 22;

// Waits, as a warp, for the phase of `parity` to end, at most `tries` times; false
// (and the CTA's abort flag) when it does not, or when another warp gave up.
// Decided by votes, so that the compiler knows that the warp stays together.
__device__ __forceinline__ bool bar_try(uint64_t* bar, int parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return __all_sync(0xFFFFFFFFu, ok);
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, int parity, volatile int* abort, int tries) {
    if (bar_try(bar, parity)) return true;
#pragma unroll 1
    for (int i = 0; i < tries; ++i) {
        if (bar_try(bar, parity)) return true;
        if (__any_sync(0xFFFFFFFFu, *abort)) return false;
    }
    *abort = 1;
    return false;
}
// 32 columns of the warp's lanes; they are there, and may be used, after the wait.
__device__ __forceinline__ void tmem_ld32(uint32_t (&x)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
        : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&x)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]), "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]), "+r"(x[21]), "+r"(x[22]), "+r"(x[23]), "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]), "+r"(x[30]), "+r"(x[31])
                 :
                 : "memory");
}

// Softmax warps, four a tile; for K and V four, or four each where steps come
// faster (one tile, or two that take turns) and the softmax does with fewer
// registers; one that issues the products. Up to sixteen warps leave 128
// registers a thread, up to twenty 96.
template <int DP>
constexpr int kSoftWarps = 4 * kChunkTiles<DP>;
template <int DP, bool SHARED>
constexpr int kCodeWarps = kChunkTiles<DP> == 1 || SHARED ? 8 : 4;
template <int DP, bool SHARED>
constexpr int kChunkThreads = 32 * (kSoftWarps<DP> + kCodeWarps<DP, SHARED> + 1);

template <int DP>
struct ChunkSmem {
    // Operand tiles of 64 x 16-bit columns, 128 bytes a row, swizzled.
    uint8_t q[kChunkTiles<DP>][DP / 64][128 * 128];
    uint8_t k[kChunkTiles<DP>][DP / 64][128 * 128];
    uint8_t v[kChunkTiles<DP>][2][DP * 128];
    float factor[kChunkTiles<DP>][128];
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], pv_done[2], done;
    uint32_t tmem;
    int abort;
};

// The same as the streaming loads, or zeros without a load; nothing waits for what is loaded.
template <int NWORDS>
__device__ __forceinline__ void load_words_if(uint32_t (&w)[NWORDS], const uint8_t* p, bool in) {
    if constexpr (NWORDS == 4) {
        const uint4 v = q8::load_stream_if(p, in);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (NWORDS == 2) {
        const uint2 v = q8::load_stream8_if(p, in);
        w[0] = v.x; w[1] = v.y;
    } else {
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.u32 p, %2, 0;\nmov.b32 %0, 0;\n@p ld.global.nc.L1::no_allocate.u32 %0, [%1];\n}\n"
            : "=&r"(w[0]) : "l"(p), "r"(static_cast<uint32_t>(in)));
    }
}
__device__ __forceinline__ uint32_t load_scale(const __half* p) {
    uint16_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_scale_if(const __half* p, bool in) {
    uint16_t v;
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %2, 0;\nmov.b16 %0, 0;\n@p ld.global.nc.L1::no_allocate.u16 %0, [%1];\n}\n"
                 : "=&h"(v) : "l"(p), "r"(static_cast<uint32_t>(in)));
    return v;
}

// SHARED: 128 rows or fewer a kv head; both tiles take the same rows and every
// other step, as two splits.
template <int DP, bool SHARED>
__global__ void __launch_bounds__(kChunkThreads<DP, SHARED>, 1) chunk_kernel(Q4Params pp) {
    using Smem = ChunkSmem<DP>;
    const q8::AttnParams& p = pp.a;
    constexpr int TILES = kChunkTiles<DP>, STAGES = TILES, ROWS = 128 * TILES;
    static_assert(!SHARED || TILES == 2, "two tiles to share rows");
    extern __shared__ uint8_t smem_raw[];
    // The swizzle counts from 1024-byte boundaries.
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + (-smem_addr(smem_raw) & 1023));
    const CacheDev& c = pp.c;
    constexpr int THREADS = kChunkThreads<DP, SHARED>, SOFT = kSoftWarps<DP>, MMA = SOFT + kCodeWarps<DP, SHARED>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = (p.R + ROWS - 1) / ROWS;
    // Later rows see more tokens: they go first.
    const int parts = SHARED ? p.nsplits / 2 : p.nsplits;  // CTAs along the tokens
    const int split = blockIdx.x % parts, r0 = (tiles - 1 - blockIdx.x / parts) * ROWS, h = blockIdx.y, b = blockIdx.z;
    const int len = q8::len_of(p, b), qlen = q8::q_len_of(p, b), rows = min(ROWS, p.R - r0);
    const int bh = b * c.H + h;
    const int64_t unit = (static_cast<int64_t>(bh) * p.nsplits + (SHARED ? 2 * split : split)) * p.R + r0;
    const int end = r0 / p.G < qlen ? q8::seen_by(p, min((r0 + rows - 1) / p.G, qlen - 1), len, qlen) : 0;
    const int t_begin = split * p.split, t_end = min(t_begin + p.split, end);
    const int steps = t_end > t_begin ? (t_end - t_begin + kChunkTokens - 1) / kChunkTokens : 0;
    if (steps == 0) {
        // Nothing to see for any row.
        for (int i = threadIdx.x; i < rows; i += THREADS) {
            if (p.nsplits > 1) {
                p.part_ml[unit + i] = make_float2(-CUDART_INF_F, 0.f);
                if (SHARED) p.part_ml[unit + p.R + i] = make_float2(-CUDART_INF_F, 0.f);
                continue;
            }
            const int64_t row = q8::out_row(p, b, h, r0 + i);
            if (p.lse_out) p.lse_out[row] = -CUDART_INF_F;
        }
        if (p.nsplits == 1)
            for (int i = threadIdx.x; i < rows * c.D; i += THREADS)
                q8::store_elem(p.out, p.out_dtype, q8::out_row(p, b, h, r0 + i / c.D) * c.D + i % c.D, 0.f);
        return;
    }

    // Steps of a tile: all, or every other one.
    const bool two = TILES == 2 && (SHARED || rows > 128);  // else the second tile rests
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&sm.k_full[i], 128);
            bar_init(&sm.v_full[i], 128);
            bar_init(&sm.k_empty[i], 1);
            bar_init(&sm.v_empty[i], 1);
            bar_init(&sm.s_full[i], 1);
            bar_init(&sm.p_full[i][0], 128);
            bar_init(&sm.p_full[i][1], 128);
            bar_init(&sm.pv_done[i], 1);
        }
        bar_init(&sm.q_full, 32 * SOFT);
        bar_init(&sm.done, 2);
        sm.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sm.tmem;

    const int tile = warp >> 2, tile_row = threadIdx.x & 127, my_row = SHARED ? tile_row : threadIdx.x;  // of a softmax thread
    int bound = 0;
    bool blind = true;
    if (warp < SOFT) {
        // A row without tokens goes along unmasked, as zeros, and is dropped at
        // the end.
        const int seen = my_row < rows ? q8::seen_by(p, (r0 + my_row) / p.G, len, qlen) : 0;
        blind = seen == 0;
        bound = blind ? INT_MAX : seen;
        // A warp's 32 query rows (16-bit here), to fp16 after a power of two.
        // DP / 8 lanes load a row, so that it is read in one piece.
        constexpr int LANES = DP / 8, AT_ONCE = 32 / LANES, ROUND = 8;
        const int64_t own = blind ? 0 : q8::q_row(p, b, h, r0 + my_row);  // (a division: once a row)
        const bool bf16 = p.q_dtype == AKV_Q_BF16;
        const int mine = lane / LANES, d = lane % LANES * 8;
#pragma unroll 1
        for (int i0 = 0; i0 < 32; i0 += AT_ONCE * ROUND) {
            uint4 raw[ROUND];
#pragma unroll
            for (int k = 0; k < ROUND; ++k) {
                const int i = i0 + AT_ONCE * k + mine;  // of the warp's rows
                raw[k] = make_uint4(0, 0, 0, 0);
                const bool sees = !__shfl_sync(0xFFFFFFFFu, blind, i);
                const uint16_t* at = static_cast<const uint16_t*>(p.q) + __shfl_sync(0xFFFFFFFFu, own, i) + d;
                if (sees && d < c.D) {
                    if (p.q_vec) {
                        raw[k] = __ldg(reinterpret_cast<const uint4*>(at));
                    } else {
                        uint32_t e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) e[j] = at[j];
                        raw[k] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < ROUND; ++k) {
                const uint32_t v[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
                uint32_t w[4], both = 0;  // the order of the magnitudes is that of their bits
#pragma unroll
                for (int j = 0; j < 4; ++j) both = __vmaxu2(both, v[j] & 0x7FFF7FFFu);
#pragma unroll
                for (int j = 1; j < LANES; j <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xFFFFFFFFu, both, j));
                const uint32_t top = max(both & 0xFFFFu, both >> 16);
                const int e = q8::row_exponent(bf16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(top))));
                const float up = q8::power_of_two(e);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float2 f = make_float2(__uint_as_float(v[j] << 16), __uint_as_float(v[j] & 0xFFFF0000u));
                    if (!bf16) f = __half22float2(*reinterpret_cast<const __half2*>(&v[j]));
                    w[j] = pack_half2(f.x * up, f.y * up);
                }
                const int r = tile_row - lane + i0 + AT_ONCE * k + mine;
                *reinterpret_cast<uint4*>(sm.q[tile][d / 64] + swizzled(r, d / 8 % 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                if (d == 0) sm.factor[tile][r] = p.c2 * q8::power_of_two(-e);
            }
        }
        fence_async();
        bar_arrive(&sm.q_full);
        __syncwarp();
    }

    if (warp < SOFT) {
        // ------------------------------------------------------------ softmax
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes
        const uint32_t s_tile = tmem + tile * 128 + lanes, o_at = tmem + 256 + tile * 128 + lanes;
        const float factor = sm.factor[tile][tile_row];
        float base = 0.f, l = 0.f;
        bool started = false, alive = true;
        const int my_steps = SHARED ? (steps + 1 - tile) / 2 : tile == 0 || two ? steps : 0;
        uint32_t pk[32];
        uint64_t sums[2], off2;
        const uint64_t f2 = pair_of(factor, factor);
        // p of 32 columns, into pk from `at` on, and their sum.
        auto weights = [&](const uint32_t (&x)[32], int at, uint64_t f, uint64_t off) {
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                float2 t = halves(fma2(pair_of(x[k], x[k + 1]), f, off));
                t.x = exp2_fast(t.x);
                t.y = exp2_fast(t.y);
                sums[k / 2 & 1] = add2(sums[k / 2 & 1], pair_of(t.x, t.y));
                pk[at + k / 2] = pack_half2(t.x, t.y);
            }
        };
        auto total = [&]() {
            const float2 both = halves(add2(sums[0], sums[1]));
            return both.x + both.y;
        };
        // The same of 64 columns where something is out of the ordinary: a row
        // that does not see all of them or has seen nothing before, scores so large that fp32
        // has no bits for differences to the base, p that leave fp16. In the
        // first and the third case S becomes t itself: -inf for what is not seen, and
        // scores that are rounded first, to the base's own multiples, so that
        // one raise is enough. (`tries` is a limit all the same.)
        auto with_care = [&](uint32_t s_at, int t0, int phase) {
            auto largest = [&](float sub, float f) {
                float m = -CUDART_INF_F;
#pragma unroll 1
                for (int g = 0; g < 4; ++g) {
                    uint32_t s[16];
                    tmem_ld16(s, s_at + 16 * g);
                    tmem_wait_ld(s);
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (t0 + 16 * g + k < bound) m = fmaxf(m, fmaf(__uint_as_float(s[k]), f, -sub));
                }
                return m;
            };
            if (__any_sync(0xFFFFFFFFu, !started)) {
                const float m = largest(0.f, factor);
                if (!started && m != -CUDART_INF_F) {
                    base = m - 6.f;
                    started = true;
                }
                __syncwarp();
            }
            float add, shift = 0.f;
            bool placed = false;  // S holds t, less `shift`, of this half
            for (int tries = 0;; ++tries) {
                if (!placed && __any_sync(0xFFFFFFFFu, t0 + kChunkHalf > bound || fabsf(base) >= 1048576.f)) {
#pragma unroll 1
                    for (int g = 0; g < 4; ++g) {
                        uint32_t s[16];
                        tmem_ld16(s, s_at + 16 * g);
                        tmem_wait_ld(s);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            s[k] = __float_as_uint(t0 + 16 * g + k < bound ? __fmul_rn(__uint_as_float(s[k]), factor) - base : -CUDART_INF_F);
                        tmem_st16(s_at + 16 * g, s);
                    }
                    tmem_wait_st();
                    placed = true;
                }
                const float f = placed ? 1.f : factor, off = placed ? -shift : -base;
                sums[0] = sums[1] = 0;
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t x[32];
                    tmem_ld32(x, s_at + 32 * g);
                    tmem_wait_ld32(x);
                    weights(x, 16 * g, pair_of(f, f), pair_of(off, off));
                }
                add = total();
                const bool over = add > 32768.f;
                if (!__any_sync(0xFFFFFFFFu, over) || tries == 8) break;
                // Some row's p may leave fp16: raise its base, scale its sums, again.
                const float m = largest(placed ? shift : base, f);
                const float up = over ? m - 6.f : 0.f;
                const float to = base + up, alpha = exp2_fast(base - to);
                shift += to - base;
                base = to;
                l *= alpha;
                if (!placed) shift = 0.f;
                if (phase > 0) {
                    // The last P V of the tile may still be running.
                    alive = bar_wait(&sm.pv_done[tile], (phase - 1) & 1, &sm.abort, pp.wait_tries);
                    if (!alive) break;
                    fence_after();
#pragma unroll 1
                    for (int g = 0; g < DP / 16; ++g) {
                        uint32_t o[16];
                        tmem_ld16(o, o_at + 16 * g);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        tmem_st16(o_at + 16 * g, o);
                    }
                }
            }
            return add;
        };
        for (int turn = 0; turn < my_steps && alive; ++turn) {
            const int t0 = t_begin + (SHARED ? 2 * turn + tile : turn) * kChunkTokens;
            alive = bar_wait(&sm.s_full[tile], turn & 1, &sm.abort, pp.wait_tries);
            if (!alive) break;
            fence_after();
            uint32_t x[32], y[32];
            constexpr bool AHEAD = THREADS <= 512;  // there are registers to load ahead into
            if (AHEAD) tmem_ld32(x, s_tile);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t s_at = s_tile + kChunkHalf * half;
                const int t = t0 + kChunkHalf * half;
                sums[0] = sums[1] = 0;
                off2 = pair_of(-base, -base);
                if constexpr (AHEAD) {
                    // Each quarter of the columns is loaded while the one before is worked on.
                    tmem_wait_ld32(x);
                    tmem_ld32(y, s_at + 32);
                    weights(x, 0, f2, off2);
                    tmem_wait_ld32(y);
                    if (half == 0) tmem_ld32(x, s_tile + kChunkHalf);
                    weights(y, 16, f2, off2);
                } else {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        tmem_ld32(x, s_at + 32 * g);
                        tmem_wait_ld32(x);
                        weights(x, 16 * g, f2, off2);
                    }
                }
                float add = total();
                if (__any_sync(0xFFFFFFFFu, !started || t + kChunkHalf > bound || fabsf(base) >= 1048576.f || add > 32768.f)) {
                    if (AHEAD && half == 0) tmem_wait_ld32(x);
                    add = with_care(s_at, t, 2 * turn + half);
                    if (!alive) break;
                }
                l += add;
#pragma unroll
                for (int g = 0; g < 2; ++g) tmem_st16(s_at + 16 * g, pk + 16 * g);
                tmem_wait_st();
                fence_before();
                bar_arrive(&sm.p_full[tile][half]);
            }
        }
        // ---------------------------------------------------------- write rows
        alive = alive && bar_wait(&sm.done, 0, &sm.abort, pp.wait_tries);
        fence_after();
        // `done` ends as well where the issuing warp gave up, some products short.
        alive = alive && !__any_sync(0xFFFFFFFFu, *static_cast<volatile int*>(&sm.abort));
        if (!alive) l = CUDART_NAN_F;  // the rows become NaN
        const bool none = alive && (blind || (!started && !isnan(l)));
        const float inv = p.nsplits > 1 ? 1.f : none ? 0.f : 1.f / l;
        const int64_t part = unit + (SHARED && tile ? p.R : 0);
        // A warp's rows go through its own part of the operands' room, which
        // nothing uses any more once all products are done, so that they are
        // written in one piece each. Pieces of 16 bytes lie crosswise. (After giving
        // up a code warp may still store there.)
        constexpr int PER = DP / 4;  // pieces of a row
        float4* const room = reinterpret_cast<float4*>(&sm.q[0][0][0]) + static_cast<int64_t>(warp) * 32 * PER;
        const int there = min(rows - (my_row - lane), 32);  // the warp's rows
        const int64_t own = my_row < rows ? q8::out_row(p, b, h, r0 + my_row) : 0;
        if (there > 0) {
#pragma unroll 1
            for (int g = 0; g < (alive ? DP / 16 : 0); ++g) {
                uint32_t o[16];
                tmem_ld16(o, o_at + 16 * g);
                tmem_wait_ld(o);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 v = none ? make_float4(0.f, 0.f, 0.f, 0.f)
                                          : make_float4(__uint_as_float(o[4 * k]) * inv, __uint_as_float(o[4 * k + 1]) * inv,
                                                        __uint_as_float(o[4 * k + 2]) * inv, __uint_as_float(o[4 * k + 3]) * inv);
                    room[lane * PER + ((4 * g + k) ^ (lane & (PER - 1)))] = v;
                }
            }
            __syncwarp();
            const int64_t mine = p.nsplits > 1 ? part + my_row : own;
            // Four pieces a lane at once, so that none waits for the one before.
            auto write = [&](auto store) {
#pragma unroll 1
                for (int m = 0; m < PER && m * 32 / PER < there; m += 4) {
                    float4 v[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int at = 32 * (m + u) + lane, r = at / PER, k = at % PER;
                        v[u] = alive ? room[r * PER + (k ^ (r & (PER - 1)))] : make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F);
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int at = 32 * (m + u) + lane, r = at / PER, k = at % PER;
                        const int64_t to = __shfl_sync(0xFFFFFFFFu, mine, r);
                        if (r < there && 4 * k < c.D) store(to * c.D + 4 * k, v[u]);
                    }
                }
            };
            if (p.nsplits > 1) write([&](int64_t at, float4 v) { *reinterpret_cast<float4*>(p.part_o + at) = v; });
            else write([&](int64_t at, float4 v) { q8::store4(p.out, p.out_dtype, at, v); });
        }
        if (my_row < rows) {
            if (p.nsplits > 1) p.part_ml[part + my_row] = make_float2(none ? -CUDART_INF_F : isnan(l) ? l : base, l);
            else if (p.lse_out)
                p.lse_out[own] = (none ? -CUDART_INF_F : isnan(l) ? l : base + log2f(l)) * 0.69314718055994531f;
        }
    } else if (warp < MMA) {
        // --------------------------------------------------- K's and V's values
        constexpr bool ALL = kCodeWarps<DP, SHARED> == 4;
        const bool does_k = ALL || warp < SOFT + 4, does_v = ALL || !does_k;
        // A lane takes pieces of 32 channels, a scale each; two or four lanes
        // a row. Eight lanes store 16 bytes each into different banks: pieces
        // of the second 64-column tile go in another order, two words ahead.
        const int tid = (threadIdx.x - 32 * SOFT) & 127;
        constexpr int LANES = DP / 32 < 4 ? DP / 32 : 4, PIECES = DP / 32 / LANES, ROWS_K = 128 / LANES;  // rows at a time, LANES times
        const int k_row = tid / LANES, k_piece = tid % LANES, turn_k = k_piece & 2;
        const uint8_t* head = c.k.codes + b * c.k.sB + h * c.k.sH;
        const __half* scales = c.k.scales + b * c.k.cB + h * c.k.cH;
        // Every step within one page: one look at the table for all its rows.
        const bool one_page = c.page_shift == 31 || (c.P % kChunkTokens == 0 && t_begin % kChunkTokens == 0);
        const int64_t rows_k = ROWS_K * c.k.sT;
        uint32_t kr[LANES][PIECES][4], ks[LANES][PIECES];
        auto piece_of = [&](int k) { return k_piece + 4 * k < c.D / 32 ? k_piece + 4 * k : 0; };
        auto load_k = [&](int t0) {
            int row = 0, phys = -1;
            if (one_page && t0 < t_end) phys = page_of(c, b, t0, row);
            const uint8_t* at = head + phys * c.k.sP + (row + k_row) * c.k.sT;
            const __half* s_at = scales + phys * c.k.cP + row + k_row;
            if (__all_sync(0xFFFFFFFFu, phys >= 0 && t0 + kChunkTokens <= t_end)) {
#pragma unroll
                for (int i = 0; i < LANES; ++i) {
#pragma unroll
                    for (int k = 0; k < PIECES; ++k) {
                        load_words(kr[i][k], at + 16 * piece_of(k));
                        ks[i][k] = load_scale(s_at + ROWS_K * i + piece_of(k) * c.k.cG);
                    }
                    at += rows_k;
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < LANES; ++i) {
                const int t = t0 + ROWS_K * i + k_row;
                if (!one_page) {
                    phys = t < t_end ? page_of(c, b, t, row) : -1;
                    at = head + phys * c.k.sP + row * c.k.sT;
                    s_at = scales + phys * c.k.cP + row;
                }
                const bool in = phys >= 0 && t < t_end;
#pragma unroll
                for (int k = 0; k < PIECES; ++k) {
                    load_words_if(kr[i][k], at + 16 * piece_of(k), in);
                    ks[i][k] = load_scale_if(s_at + piece_of(k) * c.k.cG, in);
                }
                at += rows_k;
                s_at += ROWS_K;
            }
        };
        // Eight lanes take the 64 tokens of a tile row, eight tokens each, of
        // channels that share a scale.
        const int w = warp & 3;
        constexpr int VW = DP / 64;  // words of a token per lane
        const int v_tok = 64 * (w & 1) + 8 * (lane & 7), v_d = (w >> 1) * (DP / 2) + (lane >> 3) * (DP / 8);
        const int v_from = v_d < c.D ? v_d : 0;
        const uint8_t* v_head = c.v.codes + b * c.v.sB + h * c.v.sH + v_from / 2;
        const __half* v_scales = c.v.scales + b * c.v.cB + h * c.v.cH + v_from / AKV_Q4_GROUP * c.v.cG;
        uint32_t vr[8][VW];
        uint32_t vs[4];  // scales of pairs of tokens
        auto load_v = [&](int t0) {
            const int t = t0 + v_tok;
            int row = 0;
            const int phys = t < t_end ? page_of(c, b, t, row) : -1;
            const uint8_t* at = v_head + phys * c.v.sP + row * c.v.sT;
            const __half* s_at = v_scales + phys * c.v.cP + row;  // (a page holds all of the eight tokens' scales)
            const int left = phys >= 0 ? t_end - t : 0;
            if (__all_sync(0xFFFFFFFFu, left >= 8)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    load_words(vr[i], at);
                    at += c.v.sT;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint2 s = load_scales(s_at + 4 * i);
                    vs[2 * i] = s.x;
                    vs[2 * i + 1] = s.y;
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                load_words_if(vr[i], at, i < left);
                at += c.v.sT;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint2 s = q8::load_stream8_if(s_at + 4 * i, 4 * i < left);
                vs[2 * i] = s.x;
                vs[2 * i + 1] = s.y;
            }
            // What lies past the end may hold anything.
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[i] = 2 * i + 1 < left ? vs[i] : 2 * i < left ? vs[i] & 0xFFFFu : 0u;
        };
        if (does_k) load_k(t_begin);
        if (does_v) load_v(t_begin);
        for (int j = 0; j < steps; ++j) {
            const int st = j % STAGES;
            if (does_k) {
                // The phase before a stage's first use counts as over.
                if (!bar_wait(&sm.k_empty[st], (j / STAGES & 1) ^ 1, &sm.abort, pp.wait_tries)) break;
#pragma unroll
                for (int i = 0; i < LANES; ++i)
#pragma unroll
                    for (int k = 0; k < PIECES; ++k) {
                        uint8_t* tile_k = sm.k[st][(k_piece >> 1) + 2 * k];
                        const int r = ROWS_K * i + k_row;
                        const uint32_t sc = __byte_perm(ks[i][k], 0, 0x1010);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            uint32_t x[4];
                            codes_to_half(turn_k ? kr[i][k][w ^ 2] : kr[i][k][w], x);
                            *reinterpret_cast<uint4*>(tile_k + swizzled(r, 4 * (k_piece & 1) + (w ^ turn_k))) =
                                make_uint4(mul2(x[0], sc), mul2(x[1], sc), mul2(x[2], sc), mul2(x[3], sc));
                        }
                    }
                fence_async();
                bar_arrive(&sm.k_full[st]);
                load_k(t_begin + (j + 1) * kChunkTokens);
            }
            if (does_v) {
                if (!bar_wait(&sm.v_empty[st], (j / STAGES & 1) ^ 1, &sm.abort, pp.wait_tries)) break;
                uint8_t* tile_v = sm.v[st][w & 1];
#pragma unroll
                for (int x = 0; x < VW; ++x)
#pragma unroll
                    for (int o = 0; o < 2; ++o) {  // even channels of the word, then odd ones
                        uint32_t y[4][4];  // [pair of tokens][channel]
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t u = vr[2 * q][x], z = vr[2 * q + 1][x];
                            codes_to_half(o ? ((u >> 4) & 0x0F0F0F0Fu) | (z & 0xF0F0F0F0u) : (u & 0x0F0F0F0Fu) | ((z << 4) & 0xF0F0F0F0u), y[q]);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            *reinterpret_cast<uint4*>(tile_v + swizzled(v_d + 8 * x + 2 * k + o, lane & 7)) =
                                make_uint4(mul2(y[0][k], vs[0]), mul2(y[1][k], vs[1]), mul2(y[2][k], vs[2]), mul2(y[3][k], vs[3]));
                    }
                fence_async();
                bar_arrive(&sm.v_full[st]);
                load_v(t_begin + (j + 1) * kChunkTokens);
            }
        }
    } else {
        // --------------------------------------------------------- the products
        // The whole warp goes through the loop, so that addresses stay in
        // uniform registers; one lane issues.
        constexpr uint32_t qk = mma_desc(128, kChunkTokens), pv = mma_desc(128, DP);
        constexpr uint32_t kTile = 128 * 128 / 16, kStage = DP / 64 * kTile;
        constexpr uint32_t vHalf = DP * 128 / 16, vStage = 2 * vHalf;
        const uint32_t q0 = operand_desc(sm.q), k0 = operand_desc(sm.k), v0 = operand_desc(sm.v);
        const bool lead = elect_lane();
        auto scores = [&](int tile, int st) {
            const uint32_t d = tmem + tile * 128, a = q0 + tile * kStage, x = k0 + st * kStage;
            if (lead) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const uint32_t off = k / 4 * kTile + k % 4 * 2;
                    mma_ss(d, a + off, x + off, qk, k > 0);
                }
                mma_commit(&sm.s_full[tile]);
            }
        };
        auto values = [&](int tile, int half, int st, bool add) {
            const uint32_t d = tmem + 256 + tile * 128, a = tmem + tile * 128 + half * kChunkHalf, x = v0 + st * vStage + half * vHalf;
            if (lead) {
#pragma unroll
                for (int k = 0; k < kChunkHalf / 16; ++k) mma_ts(d, a + 8 * k, x + 2 * k, pv, add || k > 0);
                mma_commit(&sm.pv_done[tile]);
            }
        };
        const int tiles_here = two ? 2 : 1;
        bool alive = bar_wait(&sm.q_full, 0, &sm.abort, pp.wait_tries);
        // A tile's first scores; with both tiles on the same rows, the
        // second tile's are those of step 1.
        for (int tile = 0; tile < tiles_here && alive; ++tile) {
            const int st = SHARED ? tile : 0;
            if (SHARED && tile >= steps) break;
            alive = bar_wait(&sm.k_full[st], 0, &sm.abort, pp.wait_tries);
            if (!alive) break;
            fence_after();
            scores(tile, st);
            if (lead && (SHARED || tile == tiles_here - 1)) mma_commit(&sm.k_empty[st]);
        }
        for (int j = 0; j < steps && alive; ++j) {
            // The step after this one of the same tiles.
            const int st = j % STAGES, next = SHARED ? j + 2 : j + 1, nx = next % STAGES, turn = SHARED ? j >> 1 : j;
            const bool more = next < steps;
            alive = bar_wait(&sm.v_full[st], j / STAGES & 1, &sm.abort, pp.wait_tries);
            if (more && !SHARED) alive = bar_wait(&sm.k_full[nx], next / STAGES & 1, &sm.abort, pp.wait_tries) && alive;
            const int i_end = SHARED ? 2 * st + 2 : 2 * tiles_here;
            for (int i = SHARED ? 2 * st : 0; i < i_end; ++i) {
                const int tile = i >> 1, half = i & 1;
                alive = alive && bar_wait(&sm.p_full[i >> 1][i & 1], turn & 1, &sm.abort, pp.wait_tries);
                if (!alive) break;
                fence_after();
                values(tile, half, st, turn > 0 || half > 0);
                if (lead && i == i_end - 1) mma_commit(&sm.v_empty[st]);
                if (!more || half == 0) continue;
                if (SHARED) {
                    alive = bar_wait(&sm.k_full[nx], next / STAGES & 1, &sm.abort, pp.wait_tries);
                    if (!alive) break;
                    fence_after();
                }
                scores(tile, nx);
                if (lead && i == i_end - 1) mma_commit(&sm.k_empty[nx]);
            }
        }
        // Also after giving up: nothing may be in flight when the tensor
        // memory is given back.
        if (lead) {
            mma_commit(&sm.done);
            bar_arrive(&sm.done);  // hands on whether the flag is set
        }
        int none = 0;
        bar_wait(&sm.done, 0, &none, kWaitTries);
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (warp == MMA) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        if (lane == 0 && sm.abort) q8::report(c.status, AKV_ERR_TIMEOUT);
    }
}

}  // namespace q4
}  // namespace akv
