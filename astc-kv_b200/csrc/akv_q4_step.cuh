// Attention of few rows (query tokens x heads of a kv head) over the 4-bit
// cache: decode steps, and any other shape sixteen rows at a time.
//
// The skeleton is the 8-bit cache's step kernel: one warp takes 16 tokens at a
// time, codes go from global memory straight into the tensor cores' registers,
// S^T = K Q^T, softmax with a loosely following base, O^T += V^T P^T, and the
// 64-token chunks of all sequences are divided evenly over one wave of CTAs.
// What four bits change:
//
//   K: lane (g, c) of a warp (g = lane / 4, c = lane % 4) loads a quarter of a
//   row, whose channels are one scale's (two with head_dim above 128): a
//   conversion turns each byte into an fp16 pair, and one multiplication by
//   the scale makes it the value, rounded to fp16 as the format says. So
//   scores need no scale, and K and V of any magnitude that fp16 holds are
//   served.
//   Tokens: the 16 rows of S may be any permutation of the tile's tokens. Row
//   2c + e is token 4c + e, row 2c + 8 + e token 4c + 2 + e: then the four tokens that a
//   lane has of V are consecutive, and one 8-byte load brings their scales.
//   V: codes of the same channel of two tokens have to be a pair. Two words
//   of eight channels become two words of byte pairs, even and odd
//   channels, by a shift and a three-input operation each; the conversion then
//   gives token pairs, and their scales multiply as a pair.
//
// Measured: 32 sequences of 32768 tokens, 32/8 heads, head_dim 128, 234 us in
// short runs with bf16 out, 5.2 TB/s or 79 % of a copy's rate; 248 us with
// fp32 out (sums rounded apart); 265 us at the power cap. One sequence of 384
// tokens, 9/3 heads: 6 us on the device. In the long ones no unit is full: a tile of 16
// tokens has 519 cycles of a quarter SM, in which 286 instructions issue
// (56 %); 66 conversions at 3.6 cycles and 64 fp16 multiplications at 2.0 take 46 % and
// 25 %, DRAM is busy 53 to 79 %. 16 ragged sequences of 283,000 tokens in all, in
// pages of 256, fp32 out: 99 us; the same tokens in equal sequences of one piece 78
// with fp16 out, of which ragged lengths add 12, pages 5 and fp32 sums 4 us. More loads in flight, Q kept in
// registers, three or five CTAs an SM changed nothing; a place in the page found
// by one comparison a tile, rows a known distance apart (DENSE) and masks only
// at the ends took 260 us to 234.
#pragma once
#include "akv_q4_loads.cuh"

namespace akv {
namespace q4 {

using q8::kShareTokens;
using q8::kStepCluster;
using q8::kStepThreads;
using q8::kStepWarps;

// Not volatile: only the numbers order products.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}

// A lane's part of a tile of 16 tokens, as loaded.
template <int DP>
struct Tile {
    static constexpr int KP = DP > 128 ? 2 : 1;      // pieces of a K row, a scale each
    static constexpr int KW = DP / 32 / KP;          // words of a piece
    static constexpr int VW = DP / 64;               // words of a V row
    uint32_t k[2][KP][KW], v[4][VW];
    uint2 ks[KP], vs;                                // scales of four tokens
};

// DP: head_dim rounded up to 64, 128 or 256; NT: groups of 8 rows; PLO: P in
// two parts; QLO: queries in two parts; TWIN, CLUSTER: see the 8-bit cache's step kernel.
// DENSE: head_dim is DP and the rows of codes follow one another. FOLDS: sums
// are put by, as with P in two parts, or where a CTA may go through too many tokens.
template <int DP, int NT, bool PLO, bool QLO, bool TWIN, bool CLUSTER, bool DENSE, bool FOLDS>
__global__ void __launch_bounds__(kStepThreads, DP == 256 || NT == 2 ? 2 : 4) step_kernel(Q4Params pp) {
    constexpr int KS = DP / 16;       // k-steps of S, d-tiles of O
    constexpr int ROWS = 8 * NT;
    constexpr int KP = Tile<DP>::KP, KW = Tile<DP>::KW, VW = Tile<DP>::VW;
    static_assert(!TWIN || (PLO && NT == 1), "twin rows carry P's second part");
    static_assert(FOLDS || !PLO, "short sums are part of P's second part");
    constexpr int TURN = 16 * kStepWarps;       // tokens from a tile to the warp's next
    constexpr bool SECOND = PLO && !TWIN;       // P's second part in products of its own
    // Tokens after which O goes to its sum in shared memory (FOLDS), which is rounded to nearest.
    constexpr int FOLD = !PLO ? q8::kStepLong : SECOND ? 1024 : 2048;
    __shared__ __align__(16) float red[kStepWarps][ROWS][DP];
    __shared__ float2 ml[kStepWarps][ROWS];
    __shared__ float row_scale[ROWS];
    __shared__ float2 piece[CLUSTER ? ROWS : 1];
    __shared__ uint2 qs[KS][NT][QLO ? 2 : 1][32];
    __shared__ q8::ShareScratch scratch;
    __shared__ float carry[FOLDS ? 2 * NT : 1][kStepThreads];

    const q8::AttnParams& p = pp.a;
    const CacheDev& c = pp.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
    const int groups = (p.R + ROWS - 1) / ROWS, units = c.H * groups;  // of a sequence
    int64_t at = 0, stop = 1;  // the next chunk of this CTA's share, its end
    int b, unit_of_b, chunk;
    const int ranks = CLUSTER ? -p.share_ctas : 1, rank = CLUSTER ? blockIdx.x % ranks : 0;
    if constexpr (CLUSTER) {
        b = blockIdx.x / ranks / units;
        unit_of_b = blockIdx.x / ranks % units;
        chunk = 0;
    } else {
        // Sequences without tokens or queries are nobody's share.
        for (int e = blockIdx.x; e < c.B; e += gridDim.x) {
            if (q8::share_chunks(p, e) > 0) continue;
            const int64_t values = static_cast<int64_t>(p.n) * p.Hq * c.D;
            for (int64_t i = 4 * threadIdx.x; i < values; i += 4 * kStepThreads)
                q8::store4(p.out, p.out_dtype, e * values + i, make_float4(0.f, 0.f, 0.f, 0.f));
            for (int i = threadIdx.x; i < p.n * p.Hq; i += kStepThreads)
                if (p.lse_out) p.lse_out[static_cast<int64_t>(e) * p.n * p.Hq + i] = -CUDART_INF_F;
        }
        const q8::Shares all = q8::count_shares(p, units, scratch);
        if (static_cast<int>(blockIdx.x) >= all.ctas) return;
        at = all.start(blockIdx.x);
        stop = all.start(blockIdx.x + 1);
        int64_t before;
        b = q8::find_sequence(p, at, units, scratch, before);
        const int n = q8::share_chunks(p, b);
        unit_of_b = static_cast<int>(q8::quotient(at - before, n));
        chunk = static_cast<int>(at - before - static_cast<int64_t>(unit_of_b) * n);
    }
    // The lane's own places in a tile. Columns past head_dim read column 0
    // instead: the query is 0 there, and such output columns are not stored.
    const int token_k = 4 * (g >> 1) + (g & 1), token_v = 4 * cc;
    int k_col[KP], k_group[KP];  // channels
#pragma unroll
    for (int j = 0; j < KP; ++j) {
        k_col[j] = 8 * KW * cc + 128 * j;
        if (k_col[j] >= c.D) k_col[j] = 0;
        k_group[j] = k_col[j] / AKV_Q4_GROUP;
    }
    const int v_col = DP / 8 * g < c.D ? DP / 8 * g : 0;
    const uint32_t k_sel = g & 1 ? 0x3232u : 0x1010u;

    for (bool first = true; at < stop; first = false) {
    const int n_chunks = q8::share_chunks(p, b);
    int n_mine;
    if constexpr (CLUSTER) {
        chunk = rank * n_chunks / ranks;
        n_mine = (rank + 1) * n_chunks / ranks - chunk;
        at = stop;
    } else {
        n_mine = static_cast<int>(min(static_cast<int64_t>(n_chunks - chunk), stop - at));
    }
    const bool whole = !CLUSTER && n_mine == n_chunks;
    const int h = unit_of_b / groups, r0 = unit_of_b % groups * ROWS;
    const int len = q8::len_of(p, b), qlen = q8::q_len_of(p, b);
    const int rows = min(ROWS, p.R - r0);
    const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (first ? 0 : 1)) * ROWS;  // where a piece of a unit goes
    const int t_begin = chunk * kShareTokens, t_end = min(t_begin + n_mine * kShareTokens, len);

    // The tile to be loaded next: its first token and pointers that move along
    // with it. Up to fast_end tiles are whole and in the same page; what comes
    // there is looked up anew. (Votes where all lanes agree anyway: the
    // compiler then keeps the warp together at no cost.)
    int t_load = t_begin + 16 * warp, fast_end = 0, left = 0;  // left: tokens of the tile that there are, 0 where it is not mapped
    bool fast = false;
    const uint8_t *k_at = nullptr, *v_at = nullptr;
    const __half *ks_at[KP], *vs_at = nullptr;
    const int64_t k_row = DENSE ? DP / 2 : c.k.sT, v_row = DENSE ? DP / 2 : c.v.sT;
    auto find_tile = [&]() {
        left = 0;
        fast_end = INT_MIN;
        fast = false;
        if (t_load >= t_end) return;
        int row;
        const int phys = page_of(c, b, t_load, row);
        if (phys < 0) return;
        left = min(t_end - t_load, 16);
        fast_end = min(t_end, t_load - row + c.P) - 15;
        fast = t_load < fast_end;
        k_at = c.k.codes + code_offset(c.k, b, h, phys, row) + token_k * k_row;
        v_at = c.v.codes + code_offset(c.v, b, h, phys, row) + token_v * v_row + v_col / 2;
#pragma unroll
        for (int j = 0; j < KP; ++j) ks_at[j] = c.k.scales + scale_offset(c.k, b, h, phys, row) + k_group[j] * c.k.cG + (token_k & ~3);
        vs_at = c.v.scales + scale_offset(c.v, b, h, phys, row) + v_col / AKV_Q4_GROUP * c.v.cG + token_v;
    };
    auto next_tile = [&]() {
        t_load += TURN;
        k_at += TURN * k_row;
        v_at += TURN * v_row;
#pragma unroll
        for (int j = 0; j < KP; ++j) ks_at[j] += TURN;
        vs_at += TURN;
        fast = __all_sync(0xFFFFFFFFu, t_load < fast_end);
        if (!fast) find_tile();
    };
    auto load_k = [&](Tile<DP>& t) {
        if (fast) {
#pragma unroll
            for (int j = 0; j < KP; ++j) {
#pragma unroll
                for (int i = 0; i < 2; ++i) load_words(t.k[i][j], k_at + 2 * i * k_row + k_col[j] / 2);
                t.ks[j] = load_scales(ks_at[j]);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < KP; ++j) {
            t.ks[j] = make_uint2(0, 0);
            if (left > 0) t.ks[j] = load_scales(ks_at[j]);  // a page's scales reach to the tile's end
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int w = 0; w < KW; ++w) t.k[i][j][w] = 0;
                if (token_k + 2 * i < left) load_words(t.k[i][j], k_at + 2 * i * k_row + k_col[j] / 2);
            }
        }
    };
    auto load_v = [&](Tile<DP>& t) {
        if (fast) {
#pragma unroll
            for (int i = 0; i < 4; ++i) load_words(t.v[i], v_at + i * v_row);
            t.vs = load_scales(vs_at);
            return;
        }
        t.vs = make_uint2(0, 0);
        const int mine = left - token_v;  // what lies past the end may hold anything: codes and scales are 0 there
        if (mine > 0) {
            t.vs = load_scales(vs_at);
            if (mine < 4) t.vs.y &= mine == 3 ? 0xFFFFu : 0u;
            if (mine < 2) t.vs.x &= 0xFFFFu;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int w = 0; w < VW; ++w) t.v[i][w] = 0;
            if (i < mine) load_words(t.v[i], v_at + i * v_row);
        }
    };

    Tile<DP> ta, tb;
    find_tile();
    load_k(ta);
    load_v(ta);
    next_tile();
    load_k(tb);
    load_v(tb);

    // Query fragments: n = g, d as in load_k.
    float factor[NT][2];   // of the lane's score columns, rows 2c and 2c + 1
    int bound[NT][2];      // tokens that those rows see (rows past the last: all)
    int bound_min = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = TWIN ? g & 3 : 8 * nt + g;
        const bool in = r < rows;
        constexpr int PER = 8 * KW;  // channels of a piece
        float x[KP][PER];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < KP; ++j) {
#pragma unroll
            for (int k = 0; k < PER; k += 16) {
                float y[16];
                if (in && PER * cc + 128 * j < c.D) {
                    q8::load_q16(p, q8::q_row(p, b, h, r0 + r) + PER * cc + 128 * j + k, y);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    x[j][k + e] = y[e];
                    top = __uint_as_float(max(__float_as_uint(top), q8::abs_bits(y[e])));
                }
            }
        }
        uint32_t tb_ = __float_as_uint(top);
        tb_ = max(tb_, __shfl_xor_sync(0xFFFFFFFFu, tb_, 1));
        tb_ = max(tb_, __shfl_xor_sync(0xFFFFFFFFu, tb_, 2));
        const int e = q8::row_exponent(__uint_as_float(tb_));
        const float up = q8::power_of_two(e);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = x[4 * s / PER][4 * s % PER + k] * up;
            const uint32_t h0 = q8::pack_half2(y[0], y[1]), h1 = q8::pack_half2(y[2], y[3]);
            if (warp == 0) {
                qs[s][nt][0][lane] = make_uint2(h0, h1);
                if (QLO) qs[s][nt][QLO ? 1 : 0][lane] = make_uint2(q8::pack_rest(y[0], y[1], h0), q8::pack_rest(y[2], y[3], h1));
            }
        }
        const float f = p.c2 * q8::power_of_two(-e);
        const int bnd = in ? q8::seen_by(p, (r0 + r) / p.G, len, qlen) : INT_MAX;
        bound_min = min(bound_min, __reduce_min_sync(0xFFFFFFFFu, bnd));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            factor[nt][k] = __shfl_sync(0xFFFFFFFFu, f, 8 * cc + 4 * k);
            bound[nt][k] = __shfl_sync(0xFFFFFFFFu, bnd, 8 * cc + 4 * k);
        }
    }
    __syncthreads();

    float o[KS][NT][4];
    float base[NT][2], limit[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < KS; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) { base[nt][k] = 0.f; limit[nt][k] = -CUDART_INF_F; l[nt][k] = 0.f; if (FOLDS) carry[2 * nt + k][threadIdx.x] = 1.f; }
    }

    auto tile = [&](int t0, Tile<DP>& t) {
        // Two sums per score: the tensor cores truncate as they add.
        float s[NT][4], s1[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[nt][k] = s1[nt][k] = 0.f;
#pragma unroll
        for (int j = 0; j < KP; ++j) {
            const uint32_t sa = __byte_perm(t.ks[j].x, 0, k_sel), sb = __byte_perm(t.ks[j].y, 0, k_sel);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                uint32_t a[4], z[4];
                codes_to_half(t.k[0][j][w], a);
                codes_to_half(t.k[1][j][w], z);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[e] = mul2(a[e], sa);
                    z[e] = mul2(z[e], sb);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int k = 2 * (j * KW + w) + e;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float(&acc)[4] = k & 1 ? s1[nt] : s[nt];
                        const uint2 q = qs[k][nt][0][lane];
                        mma(acc, a[2 * e], z[2 * e], a[2 * e + 1], z[2 * e + 1], q);
                        if (QLO) {
                            const uint2 ql = qs[k][nt][QLO ? 1 : 0][lane];
                            mma(acc, a[2 * e], z[2 * e], a[2 * e + 1], z[2 * e + 1], ql);
                        }
                    }
                }
            }
        }
        // The tile after the next one takes this one's registers.
        next_tile();
        load_k(t);

#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[nt][k] = (s[nt][k] + s1[nt][k]) * factor[nt][k & 1];
        if (__any_sync(0xFFFFFFFFu, t0 + 16 > bound_min)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (t0 + token_k + 2 * (k >> 1) >= bound[nt][k & 1]) s[nt][k] = -CUDART_INF_F;
        }
        bool above = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) above |= s[nt][k] > limit[nt][k & 1];
        if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x = fmaxf(s[nt][k], s[nt][k + 2]);
                    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
                    // The row's largest p is to be 2^8 again; rows below
                    // their limit stay as they are.
                    // (Rounded so that with large scores, too, what is below
                    // the limit is less than 16 above the base.)
                    const bool up = x > limit[nt][k];
                    const float to = up ? __fadd_ru(x, -8.f) : base[nt][k];
                    const float alpha = limit[nt][k] == -CUDART_INF_F ? 0.f : q8::exp2_fast(base[nt][k] - to);
                    base[nt][k] = to;
                    limit[nt][k] = up ? __fadd_rd(to, 15.5f) : limit[nt][k];
                    l[nt][k] *= alpha;
                    if (FOLDS) carry[2 * nt + k][threadIdx.x] *= alpha;
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        o[i][nt][k] *= alpha;
                        o[i][nt][k + 2] *= alpha;
                    }
                }
        }
        uint32_t ph[NT][2], pl[SECOND ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s[nt][k] = q8::exp2_fast(s[nt][k] - base[nt][k & 1]);
                l[nt][k & 1] += s[nt][k];
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t hi = q8::pack_half2(s[nt][2 * k], s[nt][2 * k + 1]);
                if (SECOND) pl[SECOND ? nt : 0][k] = q8::transpose8x8(q8::pack_rest(s[nt][2 * k], s[nt][2 * k + 1], hi));
                if (TWIN && cc >= 2) hi = q8::pack_rest(s[nt][2 * k], s[nt][2 * k + 1], hi);
                ph[nt][k] = q8::transpose8x8(hi);
            }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            // Channels 0, 2, 4, 6 and 1, 3, 5, 7 of the word, a byte each: two tokens.
            uint32_t even[2][4], odd[2][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t x = t.v[2 * k][w], z = t.v[2 * k + 1][w], sc = k ? t.vs.y : t.vs.x;
                codes_to_half((x & 0x0F0F0F0Fu) | ((z << 4) & 0xF0F0F0F0u), even[k]);
                codes_to_half(((x >> 4) & 0x0F0F0F0Fu) | (z & 0xF0F0F0F0u), odd[k]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    even[k][e] = mul2(even[k][e], sc);
                    odd[k][e] = mul2(odd[k][e], sc);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float(&acc)[4] = o[4 * w + e][nt];
                    mma(acc, even[0][e], odd[0][e], even[1][e], odd[1][e], make_uint2(ph[nt][0], ph[nt][1]));
                    if (SECOND) mma(acc, even[0][e], odd[0][e], even[1][e], odd[1][e], make_uint2(pl[SECOND ? nt : 0][0], pl[SECOND ? nt : 0][1]));
                }
        }
        load_v(t);
    };
    // O's sum, brought to the present base by `carry`: the lane's own part of
    // the room that `red` takes at the end.
    float4* const sums = reinterpret_cast<float4*>(&red[warp][0][0]) + lane;
    for (int t0 = t_begin + 16 * warp; __any_sync(0xFFFFFFFFu, t0 < t_end); t0 += 2 * TURN) {
        tile(t0, ta);
        if (__any_sync(0xFFFFFFFFu, t0 + TURN < t_end)) tile(t0 + TURN, tb);
        if (FOLDS && __any_sync(0xFFFFFFFFu, t0 % FOLD >= FOLD - 2 * TURN)) {
            const bool begun = t0 - t_begin >= FOLD;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float f0 = carry[2 * nt][threadIdx.x], f1 = carry[2 * nt + 1][threadIdx.x];
                carry[2 * nt][threadIdx.x] = carry[2 * nt + 1][threadIdx.x] = 1.f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    float(&x)[4] = o[i][nt];
                    float4 v = begun ? sums[(i * NT + nt) * 32] : make_float4(0.f, 0.f, 0.f, 0.f);
                    v = make_float4(fmaf(v.x, f0, x[0]), fmaf(v.y, f1, x[1]), fmaf(v.z, f0, x[2]), fmaf(v.w, f1, x[3]));
                    sums[(i * NT + nt) * 32] = v;
                    x[0] = x[1] = x[2] = x[3] = 0.f;
                }
            }
        }
    }

    q8::allow_next_kernel();
    const int begun = t_begin + 16 * warp;
    if (FOLDS && begun + (FOLD - 1 - begun % FOLD) / (32 * kStepWarps) * (32 * kStepWarps) < t_end) {  // there is a sum
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float f0 = carry[2 * nt][threadIdx.x], f1 = carry[2 * nt + 1][threadIdx.x];
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const float4 v = sums[(i * NT + nt) * 32];
                float(&x)[4] = o[i][nt];
                x[0] = fmaf(v.x, f0, x[0]); x[1] = fmaf(v.y, f1, x[1]); x[2] = fmaf(v.z, f0, x[2]); x[3] = fmaf(v.w, f1, x[3]);
            }
        }
    }
    // Join the warps in their order: (m, l) first, then O under the common maximum.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float x = l[nt][k];
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
            // A row that saw nothing has no base; NaN scores never set one.
            if (limit[nt][k] == -CUDART_INF_F) base[nt][k] = -CUDART_INF_F;
            if (isnan(x)) base[nt][k] = x;
            if (g == 0) ml[warp][8 * nt + 2 * cc + k] = make_float2(base[nt][k], x);
        }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = 8 * nt + 2 * cc + k;
            float top = ml[0][r].x;
#pragma unroll
            for (int w = 1; w < kStepWarps; ++w) top = fmaxf(top, ml[w][r].x);
            const float a = base[nt][k] == -CUDART_INF_F ? 0.f : exp2f(base[nt][k] - top);
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) red[warp][r][DP / 8 * g + 2 * i + j] = o[i][nt][k + 2 * j] * a;
        }
    if (static_cast<int>(threadIdx.x) < rows) {
        const int r = threadIdx.x;
        float top = ml[0][r].x, sum = 0.f;
#pragma unroll
        for (int w = 1; w < kStepWarps; ++w) top = fmaxf(top, ml[w][r].x);
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w)
            if (ml[w][r].x != -CUDART_INF_F) sum += ml[w][r].y * exp2f(ml[w][r].x - top);
        const bool none = top == -CUDART_INF_F && !isnan(sum);
        if (isnan(sum)) top = sum;
        row_scale[r] = none ? 0.f : 1.f / sum;
        if (CLUSTER) {
            piece[r] = make_float2(none ? -CUDART_INF_F : top, sum);
        } else if (!whole) {
            p.part_ml[part + r] = make_float2(none ? -CUDART_INF_F : top, sum);
        } else if (p.lse_out) {
            const float lse = none ? -CUDART_INF_F : top + log2f(sum);
            p.lse_out[q8::out_row(p, b, h, r0 + r)] = lse * 0.69314718055994531f;
        }
    }
    __syncthreads();
    // Four dimensions a thread, so many rows at a time.
    const int lanes = c.D / 4, row_step = kStepThreads / lanes, d = threadIdx.x % lanes * 4;
    for (int r = threadIdx.x / lanes; r < rows && static_cast<int>(threadIdx.x) < lanes * row_step; r += row_step) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w)
#pragma unroll
            for (int k = 0; k < (TWIN ? 2 : 1); ++k) {
                const float4 v = *reinterpret_cast<const float4*>(&red[w][r + 4 * k][d]);
                acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
            }
        if (CLUSTER) {
            *reinterpret_cast<float4*>(&red[0][r][d]) = acc;  // what this thread alone has read
        } else if (!whole) {
            *reinterpret_cast<float4*>(p.part_o + (part + r) * c.D + d) = acc;
        } else {
            const float f = row_scale[r];  // 0 for a row that saw nothing
            q8::store4(p.out, p.out_dtype, q8::out_row(p, b, h, r0 + r) * c.D + d,
                       f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
        }
    }
    if constexpr (CLUSTER) {
        __syncthreads();
        q8::cluster_sync();
        // Row r is finished by CTA r % ranks, its pieces in the order of the CTAs.
        for (int r = rank; r < rows; r += ranks) {
            float top = -CUDART_INF_F, sum = 0.f;
            float2 v[kStepCluster];
#pragma unroll
            for (int k = 0; k < kStepCluster; ++k) {
                v[k] = k < ranks ? q8::load_remote2(&piece[r], k) : make_float2(-CUDART_INF_F, 0.f);
                top = fmaxf(top, v[k].x);
            }
#pragma unroll
            for (int k = 0; k < kStepCluster; ++k)
                if (v[k].x != -CUDART_INF_F) sum += v[k].y * exp2f(v[k].x - top);
            const bool none = top == -CUDART_INF_F && !isnan(sum);
            const int64_t row = q8::out_row(p, b, h, r0 + r);
            if (static_cast<int>(threadIdx.x) < lanes) {
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < kStepCluster; ++k) {
                    if (v[k].x == -CUDART_INF_F) continue;
                    const float f = exp2f(v[k].x - top);
                    const float4 x = q8::load_remote4(&red[0][r][d], k);
                    acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
                    acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
                }
                const float f = none ? 0.f : 1.f / sum;
                q8::store4(p.out, p.out_dtype, row * c.D + d,
                           none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
            }
            if (threadIdx.x == 0 && p.lse_out)
                p.lse_out[row] = (none ? -CUDART_INF_F : isnan(sum) ? sum : top + log2f(sum)) * 0.69314718055994531f;
        }
        __syncthreads();
        q8::cluster_sync();  // nobody reads this CTA's memory any more
        return;
    }
    // On to the next unit.
    at += n_mine;
    chunk = 0;
    if (++unit_of_b == units) {
        unit_of_b = 0;
        do ++b;
        while (b < c.B && q8::share_chunks(p, b) == 0);
    }
    __syncthreads();
    }
}

}  // namespace q4
}  // namespace akv
