// Attention of many rows (query tokens x heads of a kv head) over the 8-bit
// cache with 16-bit outputs: prompt chunks, on the fifth-generation tensor
// cores.
//
// A CTA takes 256 rows of one kv head as two tiles of 128 and goes through a
// split of the tokens 128 at a time. Its warps have roles:
//
//   warps 0-3, 4-7  softmax of tile 0 and 1, one thread per row
//   warps 8-11      K, warps 12-15 V: codes from global memory to fp16 in
//                   shared memory (the conversion is shared by all 256 rows)
//   warp 16         one thread issues tcgen05.mma
//
// S = Q K^T (M 128 rows, N 128 tokens) and O += P V (N head_dim) accumulate
// in tensor memory: two S tiles and two O tiles fill its 512 columns. P is
// written as fp16 over its own S, 64 tokens at a time, and is the A operand of
// the second product. While one tile's softmax runs, the other tile's products
// do. The order of the issues is the order of execution, so an S that is there
// tells that the P V before it is done. (With S in two pieces of 64 tokens,
// each computed while the softmax worked on the other, the products took
// longer than that saved: from shared memory, N 64 costs what N 128 does.)
//
// Shared memory operands are K-major with the 128-byte swizzle: Q and K
// [row][d], V transposed to [d][token] (eight tokens of a d are paired by byte
// permutes in registers and stored as 16 bytes). Codes are exact in fp16, and
// 16-bit query rows after a power of two, as row_exponent says.
//
// Softmax: t = s * factor + log2 v - base per token block, p = 2^t, and the
// row sum adds p / v (see the step kernel for V's scale in the exponent).
// `base` follows the row maximum loosely: the first tokens set it so that
// their largest p is 2^6, and only a t above 15 (p would leave fp16) moves it
// and scales O, which after the first tokens hardly ever happens. Where a row
// does not see all of 64 tokens, and where scores are so large that fp32 has no
// bits for differences to the base, S is rewritten as t first, -inf for what is
// not seen.
//
// P is rounded to fp16 (2^-11 of itself at most), and O is added up by the
// tensor cores, which truncate: 6e-9 of it per token of the split.
//
// With head_dim above 128 a CTA has one tile of rows, one stage of K and V, and
// four warpgroups: K is warps 4-7, V 8-11, the issuing warp 12.
//
// Per step and tile the tensor cores need 1024 cycles (D = 128) and the
// special-function units as many for the 128 x 128 exp2. Measured, 2048 query
// tokens at the end of 32768, 32/8 heads, D 128: int8 1.17 ms = 917 TFLOP/s,
// 55 % of the 1657 that a large library product reaches (e4m3 1.12 ms; 1.25 ms
// int8 under the power cap). In a capture of 1024 query tokens at the end of
// 16384 the tensor pipe is active 39 % of the time; at D 256, 512 at the end of
// 8192 (223 us, 597 TFLOP/s), 26 %. What bounds it is the latency of a tile's round (scores, softmax, P, values: some
// 4500 cycles, two tiles in turn), not a unit's throughput. On the way: stalls
// on the converters' loads 2.2 to 1.43 ms, uniform issue of the products and
// separate K and V groups 1.31, S in one piece 1.17; four 16-column loads of S
// in a row instead of one ahead of the other cost 20 %.
#pragma once
#include "akv_q8_attend.cuh"

namespace akv {
namespace q8 {

// A CTA's tiles of 128 rows and its stages of K and V: with head_dim above 128
// one O tile fills half of the tensor memory, and one stage the shared memory.
template <int DP>
constexpr int kChunkTiles = DP <= 128 ? 2 : 1;
constexpr int kChunkTokens = 128;  // per step
constexpr int kChunkHalf = 64;     // P goes to the tensor cores in two parts
// Five warpgroups, whose last three warps only give their registers away; with
// one tile four, of 128 registers a thread.
template <int DP>
constexpr int kChunkThreads = 32 * (kChunkTiles<DP> == 2 ? 20 : 16);
constexpr int kMetaSlots = 4;      // K may be written three steps ahead of a softmax

template <int DP>
struct ChunkSmem {
    // Operand tiles of 64 x 16-bit columns, 128 bytes a row, swizzled.
    uint8_t q[kChunkTiles<DP>][DP / 64][128 * 128];
    uint8_t k[kChunkTiles<DP>][DP / 64][128 * 128];
    uint8_t v[kChunkTiles<DP>][2][DP * 128];
    float4 meta[kMetaSlots][kChunkTokens / 16];  // K's scale, log2 and reciprocal of V's, for 16 tokens
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], pv_done[2], done;
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Waits for the phase of `parity` to end, a bounded number of times (a try takes
// about 1.5 us, all some 6 s); false (and the CTA's abort flag) when it does
// not, or when another warp gave up.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, int parity, volatile int* abort) {
    for (int i = 0; i < 1 << 22; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if (*abort) return false;
    }
    *abort = 1;
    return false;
}

// Low word of the descriptor of a K-major operand with the 128-byte swizzle:
// its address in units of 16 bytes. The high word is the same for all: rows of
// 128 bytes, groups of eight rows 1024 bytes apart, descriptor version 1.
__device__ __forceinline__ uint32_t operand_desc(const void* p) { return (smem_addr(p) & 0x3FFFF) >> 4 | 1u << 16; }
// kind::f16 with fp16 operands, fp32 accumulation, both K-major.
__device__ __forceinline__ constexpr uint32_t mma_desc(int m, int n) {
    return 1u << 4 | static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.u32 p, %4, 0;\nmov.b64 x, {%1, 0x40004040};\nmov.b64 y, {%2, 0x40004040};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(desc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.u32 p, %4, 0;\nmov.b64 y, {%2, 0x40004040};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(desc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ bool elect_lane() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
// The barrier's phase ends when every MMA issued so far has finished.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&x)[16], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]),
          "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
        : "r"(at) : "memory");
}
// Ends the loads in flight; x is one of them and must not be used before.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&x)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]),
                   "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* x) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(x[0]),
        "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]),
        "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float2 halves(uint64_t v) {
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
    return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Byte offset of 16-byte chunk c of row r in a swizzled tile.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// SHARED: 128 rows or fewer a kv head; both tiles take the same rows and every
// other step, as two splits.
template <int FMT, int DP, bool SHARED>
__global__ void __launch_bounds__(kChunkThreads<DP>, 1) chunk_kernel(AttnParams p) {
    using Smem = ChunkSmem<DP>;
    constexpr int TILES = kChunkTiles<DP>, STAGES = TILES, ROWS = 128 * TILES;
    static_assert(!SHARED || TILES == 2, "two tiles to share rows");
    extern __shared__ uint8_t smem_raw[];
    // The swizzle counts from 1024-byte boundaries.
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + (-smem_addr(smem_raw) & 1023));
    const CacheDev& c = p.c;
    // With one tile there is no second group of softmax warps.
    constexpr int THREADS = kChunkThreads<DP>, MISSING = TILES == 2 ? 0 : 4;
    const int hw_warp = threadIdx.x >> 5, warp = hw_warp < 4 ? hw_warp : hw_warp + MISSING, lane = threadIdx.x & 31;
    const int tiles = (p.R + ROWS - 1) / ROWS;
    // Later rows see more tokens: they go first.
    const int parts = SHARED ? p.nsplits / 2 : p.nsplits;  // CTAs along the tokens
    const int split = blockIdx.x % parts, r0 = (tiles - 1 - blockIdx.x / parts) * ROWS, h = blockIdx.y, b = blockIdx.z;
    const int len = len_of(p, b), qlen = q_len_of(p, b), rows = min(ROWS, p.R - r0);
    const int bh = b * c.H + h;
    const int64_t unit = (static_cast<int64_t>(bh) * p.nsplits + (SHARED ? 2 * split : split)) * p.R + r0;
    const int end = r0 / p.G < qlen ? seen_by(p, min((r0 + rows - 1) / p.G, qlen - 1), len, qlen) : 0;
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
            const int64_t row = out_row(p, b, h, r0 + i);
            if (p.lse) p.lse[row] = -CUDART_INF_F;
            if (p.lse_out) p.lse_out[row] = -CUDART_INF_F;
        }
        if (p.nsplits == 1)
            for (int i = threadIdx.x; i < rows * c.D; i += THREADS)
                store_elem(p.out, p.out_dtype, out_row(p, b, h, r0 + i / c.D) * c.D + i % c.D, 0.f);
        return;
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&sm.k_full[i], 128);
            bar_init(&sm.v_full[i], 128);
            bar_init(&sm.k_empty[i], 1);
            bar_init(&sm.v_empty[i], 1);
            bar_init(&sm.pv_done[i], 1);
            bar_init(&sm.s_full[i], 2);
            bar_init(&sm.p_full[i][0], 128);
            bar_init(&sm.p_full[i][1], 128);
        }
        bar_init(&sm.done, 1);
        sm.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // Query rows: thread = row, to fp16 after a power of two.
    float factor = 0.f;
    int bound = 0;
    bool blind = true;
    if (warp < 4 * TILES) {
        const int tile = warp >> 2, r = threadIdx.x & 127, at_row = SHARED ? r : threadIdx.x, row = r0 + at_row;
        // A row without tokens goes along unmasked, as zeros, and is dropped at
        // the end.
        const int seen = at_row < rows ? seen_by(p, row / p.G, len, qlen) : 0;
        const bool in = seen > 0;
        const int64_t at = in ? q_row(p, b, h, row) : 0;
        uint32_t top = 0;
        if (in) {
#pragma unroll 4
            for (int d = 0; d < c.D; d += 16) {
                float x[16];
                load_q16(p, at + d, x);
#pragma unroll
                for (int k = 0; k < 16; ++k) top = max(top, abs_bits(x[k]));
            }
        }
        const int e = row_exponent(__uint_as_float(top));
        const float up = power_of_two(e);
#pragma unroll 4
        for (int d = 0; d < DP; d += 16) {
            float x[16];
            if (in && d < c.D) {
                load_q16(p, at + d, x);  // from L1
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint4 w;
                w.x = pack_half2(x[8 * k] * up, x[8 * k + 1] * up);
                w.y = pack_half2(x[8 * k + 2] * up, x[8 * k + 3] * up);
                w.z = pack_half2(x[8 * k + 4] * up, x[8 * k + 5] * up);
                w.w = pack_half2(x[8 * k + 6] * up, x[8 * k + 7] * up);
                *reinterpret_cast<uint4*>(sm.q[tile][d / 64] + swizzled(r, d / 8 % 8 + k)) = w;
            }
        }
        factor = p.c2 * power_of_two(-e);
        blind = !in;
        bound = blind ? INT_MAX : seen;
        fence_async();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sm.tmem;

    // Steps of a tile: all, or every other one.
    const bool two = TILES == 2 && (SHARED || rows > 128);  // else the second tile rests
    // Registers go to where they are needed: 2 x 136 + 2 x 80 + 48 = 5 x 96
    // (with one tile all have what they need).
    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        if (TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        const int tile = warp >> 2;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes
        const uint32_t s_tile = tmem + tile * 128 + lanes, o_at = tmem + 256 + tile * 128 + lanes;
        float base = 0.f, l = 0.f;
        bool started = false;
        bool alive = true;
        const int my_steps = SHARED ? (steps + 1 - tile) / 2 : tile == 0 || two ? steps : 0;
        for (int i = 0; i < 2 * my_steps && alive; ++i) {
            const int turn = i >> 1, half = i & 1, j = SHARED ? 2 * turn + tile : turn;
            const int t0 = t_begin + j * kChunkTokens + half * kChunkHalf;
            const float4* meta = sm.meta[j % kMetaSlots] + 4 * half;
            const uint32_t s_at = s_tile + kChunkHalf * half;
            if (half == 0) {
                alive = __all_sync(0xFFFFFFFFu, bar_wait(&sm.s_full[tile], turn & 1, &sm.abort));
                if (!alive) break;
                fence_after();
            }
            if (__any_sync(0xFFFFFFFFu, !started)) {
                // The largest t of the row's tokens.
                float m = -CUDART_INF_F;
#pragma unroll 1
                for (int g = 0; g < 4; ++g) {
                    uint32_t s[16];
                    tmem_ld16(s, s_at + 16 * g);
                    const float4 mt = meta[g];
                    tmem_wait_ld(s);
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (t0 + 16 * g + k < bound) m = fmaxf(m, fmaf(__uint_as_float(s[k]), factor * mt.x, mt.y));
                }
                if (!started && m != -CUDART_INF_F) {
                    base = m - 6.f;
                    started = true;
                }
                __syncwarp();
            }
            uint32_t pk[32];
            float add, shift = 0.f;
            bool placed = false;  // S holds t, less `shift`, of this half
            for (int tries = 0;; ++tries) {
                // Where a row does not see every token, or has a base without
                // the bits to bring an exact score within 15 of it, S becomes t
                // itself: -inf for what is not seen, and scores that are
                // rounded first, to the base's own multiples, so that one raise
                // is enough to bring them below 15. (`tries` is a limit all the same.)
                if (!placed && __any_sync(0xFFFFFFFFu, t0 + kChunkHalf > bound || fabsf(base) >= 1048576.f)) {
#pragma unroll 1
                    for (int g = 0; g < 4; ++g) {
                        uint32_t s[16];
                        tmem_ld16(s, s_at + 16 * g);
                        const float4 mt = meta[g];
                        tmem_wait_ld(s);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            s[k] = __float_as_uint(t0 + 16 * g + k < bound ? fmaf(__uint_as_float(s[k]), factor * mt.x, mt.y) - base : -CUDART_INF_F);
                        tmem_st16(s_at + 16 * g, s);
                    }
                    tmem_wait_st();
                    placed = true;
                }
                float m = -CUDART_INF_F;
                add = 0.f;
                uint32_t s[2][16];
                tmem_ld16(s[0], s_at);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t(&x)[16] = s[g & 1];
                    tmem_wait_ld(x);
                    if (g < 3) tmem_ld16(s[(g + 1) & 1], s_at + 16 * (g + 1));
                    const float4 mt = meta[g];
                    const float f = placed ? 1.f : factor * mt.x, off = placed ? -shift : mt.y - base;
                    const uint64_t f2 = pair_of(f, f), off2 = pair_of(off, off);
                    uint64_t sum = 0;
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        float2 t = halves(fma2(pair_of(x[k], x[k + 1]), f2, off2));
                        m = fmaxf(m, fmaxf(t.x, t.y));
                        t.x = exp2_fast(t.x);
                        t.y = exp2_fast(t.y);
                        sum = add2(sum, pair_of(t.x, t.y));
                        pk[8 * g + k / 2] = pack_half2(t.x, t.y);
                    }
                    const float2 both = halves(sum);
                    add = fmaf(both.x + both.y, mt.z, add);
                }
                if (!__any_sync(0xFFFFFFFFu, m > 15.f) || tries == 8) break;
                // Some row's p leaves fp16: raise its base, scale its sums, again.
                const float up = m > 15.f ? m - 6.f : 0.f;
                const float to = base + up, alpha = exp2_fast(base - to);
                shift += to - base;
                base = to;
                l *= alpha;
                if (!placed) shift = 0.f;
                if (i > 0) {
                    // The last P V of the tile may still be running.
                    alive = __all_sync(0xFFFFFFFFu, bar_wait(&sm.pv_done[tile], (i - 1) & 1, &sm.abort));
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
            l += add;
#pragma unroll
            for (int g = 0; g < 2; ++g) tmem_st16(s_at + 16 * g, pk + 16 * g);
            tmem_wait_st();
            fence_before();
            bar_arrive(&sm.p_full[tile][half]);
        }
        // ---------------------------------------------------------- write rows
        alive = __all_sync(0xFFFFFFFFu, alive && bar_wait(&sm.done, 0, &sm.abort));
        fence_after();
        const int my_row = SHARED ? threadIdx.x & 127 : threadIdx.x;
        const bool in = my_row < rows;
        const int r = r0 + my_row;
        const int64_t part = unit + my_row + (SHARED && tile ? p.R : 0);
        if (!alive) l = CUDART_NAN_F;  // gave up: the rows become NaN
        const bool none = alive && (blind || (!started && !isnan(l)));
        const float inv = none ? 0.f : 1.f / l;
        const int64_t row = in ? out_row(p, b, h, r) : 0;
#pragma unroll 1
        for (int g = 0; g < DP / 16; ++g) {
            uint32_t o[16];
            tmem_ld16(o, o_at + 16 * g);
            tmem_wait_ld(o);
            if (!in || 16 * g >= c.D) {
            } else if (p.nsplits > 1) {
                uint4* to = reinterpret_cast<uint4*>(p.part_o + part * c.D + 16 * g);
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            } else {
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float x = none ? 0.f : __uint_as_float(o[2 * k]) * inv, y = none ? 0.f : __uint_as_float(o[2 * k + 1]) * inv;
                    if (p.out_dtype == AKV_Q_BF16) {
                        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
                        w[k] = *reinterpret_cast<const uint32_t*>(&v);
                    } else {
                        w[k] = pack_half2(x, y);
                    }
                }
                uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * c.D + 16 * g);
                to[0] = make_uint4(w[0], w[1], w[2], w[3]);
                to[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
            __syncwarp();
        }
        if (in) {
            if (p.nsplits > 1) {
                p.part_ml[part] = make_float2(none ? -CUDART_INF_F : isnan(l) ? l : base, l);
            } else {
                const float lse = none ? -CUDART_INF_F : isnan(l) ? l : base + log2f(l);
                if (p.lse) p.lse[row] = lse;
                if (p.lse_out) p.lse_out[row] = lse * 0.69314718055994531f;
            }
        }
    } else if (warp < 12) {
        // ---------------------------------------------------------- K to fp16
        if (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // Four lanes a row of a 64-column tile, 32 rows at a time: the stores
        // of eight lanes (two rows, every other chunk) fall into different
        // banks.
        const int tid = threadIdx.x - 32 * (8 - MISSING);
        constexpr int KP = DP / 16;  // 16-byte pieces per lane and step
        const int k_row = tid >> 2, k_piece = tid & 3;
        int k_col[DP / 64];
#pragma unroll
        for (int i = 0; i < DP / 64; ++i) k_col[i] = 64 * i + 16 * k_piece < c.D ? 64 * i + 16 * k_piece : 0;
        const uint8_t* head = c.k.codes + b * c.k.sB + h * c.k.sH;
        const int blk_shift = 31 - __clz(c.blk);
        // Every step within one page: one look at the table for all its rows.
        const bool one_page = c.page_shift == 31 || (c.P % kChunkTokens == 0 && t_begin % kChunkTokens == 0);
        const int64_t row32 = 32 * c.k.sT;
        uint4 kr[KP];
        auto load_k = [&](int t0) {
            if (one_page) {
                int row = 0;
                const int phys = t0 < t_end ? page_of(c, b, t0, row) : -1;
                const uint8_t* at = head + phys * c.k.sP + (row + k_row) * c.k.sT;
                const int left = phys >= 0 ? t_end - t0 - k_row : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int k = 0; k < DP / 64; ++k) kr[4 * k + i] = load_stream_if(at + k_col[k], 32 * i < left);
                    at += row32;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = t0 + 32 * i + k_row;
                    int row = 0;
                    const int phys = t < t_end ? page_of(c, b, t, row) : -1;
#pragma unroll
                    for (int k = 0; k < DP / 64; ++k)
                        kr[4 * k + i] = load_stream_if(head + phys * c.k.sP + row * c.k.sT + k_col[k], phys >= 0);
                }
            }
        };
        // Read now, looked at when the step comes.
        float ks = 0.f, vs = 0.f;
        auto load_meta = [&](int t0) {
            const int t = t0 + 16 * tid;
            ks = 0.f;
            vs = 1.f;
            if (tid >= 8 || t >= t_end) return;
            int row;
            const int phys = page_of(c, b, t, row);
            if (phys < 0) return;
            ks = __ldg(c.k.scales + scale_offset(c.k, b, h, phys, row >> blk_shift));
            vs = __ldg(c.v.scales + scale_offset(c.v, b, h, phys, row >> blk_shift));
        };
        load_meta(t_begin);
        load_k(t_begin);
        for (int j = 0; j < steps; ++j) {
            const int st = j % STAGES;
            // The phase before a stage's first use counts as over.
            if (!bar_wait(&sm.k_empty[st], (j / STAGES & 1) ^ 1, &sm.abort)) break;
            if (tid < 8) {
                // A NaN scale stays one in lv, for rows that see it, and not in
                // the reciprocal, which all rows' sums take.
                const float lv = log2_fast(vs < 8.0779357e-28f ? 8.0779357e-28f : vs);
                sm.meta[j % kMetaSlots][tid] = make_float4(ks, lv, isnan(lv) ? 0.f : exp2_fast(-lv), 0.f);
            }
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                uint8_t* tile = sm.k[st][i / 4];
                const int r = 32 * (i & 3) + k_row;
                uint4 x, y;
                codes_to_half<FMT>(kr[i].x, x.x, x.y);
                codes_to_half<FMT>(kr[i].y, x.z, x.w);
                codes_to_half<FMT>(kr[i].z, y.x, y.y);
                codes_to_half<FMT>(kr[i].w, y.z, y.w);
                *reinterpret_cast<uint4*>(tile + swizzled(r, 2 * k_piece)) = x;
                *reinterpret_cast<uint4*>(tile + swizzled(r, 2 * k_piece + 1)) = y;
            }
            fence_async();
            bar_arrive(&sm.k_full[st]);
            load_meta(t_begin + (j + 1) * kChunkTokens);
            load_k(t_begin + (j + 1) * kChunkTokens);
        }
    } else if (warp < 16) {
        // ---------------------------------------------------------- V to fp16
        if (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // Eight lanes take the 64 tokens of a tile row, eight tokens each.
        const int w = warp & 3;
        constexpr int VW = DP / 32;  // words of a token per lane
        const int v_tok = 64 * (w & 1) + 8 * (lane & 7), v_d = (w >> 1) * (DP / 2) + (lane >> 3) * (DP / 8);
        const uint8_t* head = c.v.codes + b * c.v.sB + h * c.v.sH + (v_d < c.D ? v_d : 0);
        const int next16 = v_d + 16 < c.D ? 16 : 0;  // of 32 bytes a lane the second half
        uint32_t vr[8][VW];
        auto load_v = [&](int t0) {
            const int t = t0 + v_tok;
            int row = 0;
            const int phys = t < t_end ? page_of(c, b, t, row) : -1;
            const uint8_t* at = head + phys * c.v.sP + row * c.v.sT;
            const int left = phys >= 0 ? t_end - t : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (DP == 64) {
                    const uint2 x = load_stream8_if(at, i < left);
                    vr[i][0] = x.x; vr[i][1] = x.y;
                } else {
                    const uint4 x = load_stream_if(at, i < left);
                    vr[i][0] = x.x; vr[i][1] = x.y; vr[i][VW > 2 ? 2 : 0] = x.z; vr[i][VW > 2 ? 3 : 1] = x.w;
                }
                if (DP == 256) {
                    const uint4 x = load_stream_if(at + next16, i < left);
                    vr[i][VW - 4 > 0 ? VW - 4 : 0] = x.x; vr[i][VW - 3 > 0 ? VW - 3 : 0] = x.y; vr[i][VW - 2] = x.z; vr[i][VW - 1] = x.w;
                }
                at += c.v.sT;
            }
        };
        load_v(t_begin);
        for (int j = 0; j < steps; ++j) {
            const int st = j % STAGES;
            if (!bar_wait(&sm.v_empty[st], (j / STAGES & 1) ^ 1, &sm.abort)) break;
            uint8_t* tile = sm.v[st][w & 1];
#pragma unroll
            for (int x = 0; x < VW; ++x) {
                uint32_t y[4][4];  // [d of the word][pair of tokens]
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t u = vr[2 * q][x], z = vr[2 * q + 1][x];
                    codes_to_half<FMT>(__byte_perm(u, z, 0x5140), y[0][q], y[1][q]);
                    codes_to_half<FMT>(__byte_perm(u, z, 0x7362), y[2][q], y[3][q]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<uint4*>(tile + swizzled(v_d + 4 * x + k, lane & 7)) = make_uint4(y[k][0], y[k][1], y[k][2], y[k][3]);
            }
            fence_async();
            bar_arrive(&sm.v_full[st]);
            load_v(t_begin + (j + 1) * kChunkTokens);
        }
    } else {
        // --------------------------------------------------------- the products
        if (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 16) {
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
                    bar_arrive(&sm.s_full[tile]);  // hands on what k_full has shown: the block scales
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
            bool alive = true;
            // A tile's first scores; with both tiles on the same rows, the
            // second tile's are those of step 1.
            for (int tile = 0; tile < tiles_here && alive; ++tile) {
                const int st = SHARED ? tile : 0;
                if (SHARED && tile >= steps) break;
                alive = __all_sync(0xFFFFFFFFu, bar_wait(&sm.k_full[st], 0, &sm.abort));
                if (!alive) break;
                fence_after();
                scores(tile, st);
                if (lead && (SHARED || tile == tiles_here - 1)) mma_commit(&sm.k_empty[st]);
            }
            for (int j = 0; j < steps && alive; ++j) {
                // The step after this one of the same tiles.
                const int st = j % STAGES, next = SHARED ? j + 2 : j + 1, nx = next % STAGES, turn = SHARED ? j >> 1 : j;
                const bool more = next < steps;
                alive = bar_wait(&sm.v_full[st], j / STAGES & 1, &sm.abort);
                if (more && !SHARED) alive = bar_wait(&sm.k_full[nx], next / STAGES & 1, &sm.abort) && alive;
                const int i_end = SHARED ? 2 * st + 2 : 2 * tiles_here;
                for (int i = SHARED ? 2 * st : 0; i < i_end; ++i) {
                    const int tile = i >> 1, half = i & 1;
                    alive = __all_sync(0xFFFFFFFFu, alive && bar_wait(&sm.p_full[tile][half], turn & 1, &sm.abort));
                    if (!alive) break;
                    fence_after();
                    values(tile, half, st, turn > 0 || half > 0);
                    if (lead && i == i_end - 1) mma_commit(&sm.v_empty[st]);
                    if (!more || half == 0) continue;
                    if (SHARED) {
                        alive = __all_sync(0xFFFFFFFFu, bar_wait(&sm.k_full[nx], next / STAGES & 1, &sm.abort));
                        if (!alive) break;
                        fence_after();
                    }
                    scores(tile, nx);
                    if (lead && i == i_end - 1) mma_commit(&sm.k_empty[nx]);
                }
            }
            // Also after giving up: nothing may be in flight when the tensor
            // memory is given back.
            if (lead) mma_commit(&sm.done);
            int none = 0;
            bar_wait(&sm.done, 0, &none);
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (warp == 16) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        if (lane == 0 && sm.abort) report(c.status, AKV_ERR_TIMEOUT);
    }
}

}  // namespace q8
}  // namespace akv
