// Attention of few rows (query tokens x heads of a kv head) over the 8-bit
// cache: decode steps, and any other shape sixteen rows at a time.
//
// Every K and V byte of the cache is read once per group of 8 or 16 rows, so
// a decode step is bound by HBM. One warp takes 16 tokens at a time; the
// codes go from global memory straight into the registers that the tensor
// cores read, no shared memory between. That works because the contracted
// index of a matrix product may be permuted freely if both operands agree:
//
//   S^T = K Q^T (m = token, n = row, k = d): lane (g, c) of m16n8k16 (g =
//   lane / 4, c = lane % 4) holds d-groups c of tokens g and g + 8. It loads
//   16 consecutive bytes of each of these rows, and the query fragments
//   take their d in the same order.
//   O^T += V^T P^T (m = d, n = row, k = token): the lane holds tokens 2c,
//   2c + 1, 2c + 8, 2c + 9 for its own d. It loads 16 consecutive bytes of
//   these four rows (eight lanes cover a row), pairs tokens by byte permutes,
//   and the output's d follow: fragment row g of tile i is byte 2i of lane
//   group g's bytes, row g + 8 is byte 2i + 1.
//
// Codes are exact in fp16; a 16-bit query row is after a power of two, as
// row_exponent says (fp32 queries go in two parts); the block scale of K and the power go to the
// fp32 score. V's block scale v is folded into the exponent: P' = 2^(s +
// log2 v - m) and the row sum adds P' / v, so V needs no product. P' is
// scaled to between 2^8 and 2^15.5 to use fp16's range; fp32 outputs carry it
// in two fp16 parts.
// `m` follows the row maximum loosely: a score that would take P' past fp16
// raises it so that the largest P' is 2^8 again. A vote finds such scores;
// after the first tiles they are rare.
//
// The tensor cores truncate as they add, which makes a long sum smaller than it
// is. With fp32 outputs O is added, rounded to nearest, to a sum that waits in
// shared memory, every 32 products (30010 tokens by one CTA, D 256: 1.6e-5 off
// without that, of it 1.3e-5 too small, now 9e-7).
//
// The work, 64-token chunks of every (sequence, kv head, group of rows), is
// divided evenly over the CTAs of one wave, whatever the lengths: a CTA's
// share may start and end inside a unit, whose pieces the combine kernel adds
// up. (Splits of one length left CTAs idle behind the longest sequence: five
// drafted tokens over eight sequences of 205 to 8192 tokens 84 us, with even
// shares 72; what came after made it 51.)
//
// Measured (fp32 out, head_dim 128, 32/8 heads, B32, 32768 tokens: 2.15 GB):
// int8 355 us = 6.05 TB/s, 94 % of a copy's 6.42 TB/s; e4m3 336 us; under the
// power cap int8 401 us at 1.6 GHz. 402 warp instructions per 16 tokens, of
// them 176 to turn codes into fp16; issue slots 54 % used, tensor pipe 16 % (B8).
// (Without the sum in shared memory 348, 331 and 396 us.)
// What carried it there from 587 us: pointers that advance instead of index
// arithmetic (587 to 398), query fragments in shared memory rather than
// registers (398 to 385), V loaded a tile ahead (385 to 365), even shares.
#pragma once
#include "akv_q8_attend.cuh"
#include "akv_q8_step_launch.h"

namespace akv {
namespace q8 {

constexpr int kStepThreads = 32 * kStepWarps;
static_assert(kShareTokens == 16 * kStepWarps, "a tile of 16 tokens for each warp");

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// `p`, a place in this CTA's shared memory, in that of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_addr(const void* p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    return a;
}
__device__ __forceinline__ float2 load_remote2(const void* p, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_remote4(const void* p, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote_addr(p, rank)) : "memory");
    return v;
}

// TWIN (with PLO, four rows or fewer): rows 4 to 7 are rows 0 to 3 again; their
// P is the second part, so that one product does both. The power that the
// products draw slows the clock: B32, 32768 tokens int8, run for seconds at the
// 1000 W power cap, 402 us against 410 (349 against 345 in short runs).
// CLUSTER: up to eight CTAs divide one unit and add up its pieces through
// distributed shared memory; for little work, where the scan of the lengths and a second
// launch would cost more than an even division saves (B1, 384 tokens, 9/3
// heads: 8.2 us against 12.3; B8, 1024 tokens, 32/8 heads: 15.7 against 24.8).
// DP: head_dim rounded up to 64, 128 or 256; NT: groups of 8 rows; PLO: P in
// two parts; QLO: queries in two parts.
template <int FMT, int DP, int NT, bool PLO, bool QLO, bool TWIN, bool CLUSTER>
__global__ void __launch_bounds__(kStepThreads, DP == 256 || NT == 2 ? 2 : 4) step_kernel(AttnParams p) {
    constexpr int KS = DP / 16;       // k-steps of S, d-tiles of O
    constexpr int VW = DP / 32;       // words of a V row per lane
    constexpr int ROWS = 8 * NT;
    __shared__ __align__(16) float red[kStepWarps][ROWS][DP];
    __shared__ float2 ml[kStepWarps][ROWS];
    __shared__ float row_scale[ROWS];
    __shared__ float2 piece[CLUSTER ? ROWS : 1];
    __shared__ uint2 qs[KS][NT][QLO ? 2 : 1][32];

    __shared__ ShareScratch scratch;
    __shared__ float carry[PLO ? 2 * NT : 1][kStepThreads];

    const CacheDev& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
    static_assert(!TWIN || (PLO && NT == 1), "twin rows carry P's second part");
    constexpr bool SECOND = PLO && !TWIN;  // P's second part in products of its own
    constexpr int FOLD = SECOND ? 1024 : 2048;  // tokens after which O goes to its sum in shared memory (fp32 outputs)
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
            if (share_chunks(p, e) > 0) continue;
            const int64_t values = static_cast<int64_t>(p.n) * p.Hq * c.D;
            for (int64_t i = 4 * threadIdx.x; i < values; i += 4 * kStepThreads)
                store4(p.out, p.out_dtype, e * values + i, make_float4(0.f, 0.f, 0.f, 0.f));
            for (int i = threadIdx.x; i < p.n * p.Hq; i += kStepThreads) {
                const int64_t row = static_cast<int64_t>(e) * p.n * p.Hq + i;
                if (p.lse) p.lse[row] = -CUDART_INF_F;
                if (p.lse_out) p.lse_out[row] = -CUDART_INF_F;
            }
        }
        const Shares all = count_shares(p, units, scratch);
        if (static_cast<int>(blockIdx.x) >= all.ctas) return;
        at = all.start(blockIdx.x);
        stop = all.start(blockIdx.x + 1);
        int64_t before;
        b = find_sequence(p, at, units, scratch, before);
        const int n = share_chunks(p, b);
        unit_of_b = static_cast<int>(quotient(at - before, n));
        chunk = static_cast<int>(at - before - static_cast<int64_t>(unit_of_b) * n);
    }
    for (bool first = true; at < stop; first = false) {
    const int n_chunks = share_chunks(p, b);
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
    const int len = len_of(p, b), qlen = q_len_of(p, b);
    const int rows = min(ROWS, p.R - r0);
    const int bh = b * c.H + h;
    const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (first ? 0 : 1)) * ROWS;  // where a piece of a unit goes
    const int t_begin = chunk * kShareTokens, t_end = min(t_begin + n_mine * kShareTokens, len);

    // The lane's own places in a tile. Columns past head_dim read column 0
    // instead: the query is 0 there, and such output columns are not stored.
    int k_col[DP / 64], v_col[DP > 128 ? 2 : 1];
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) k_col[j] = 16 * cc + 64 * j < c.D ? 16 * cc + 64 * j : 0;
    if (DP == 64) {
        v_col[0] = 8 * g < c.D ? 8 * g : 0;
    } else {
#pragma unroll
        for (int j = 0; j < DP / 128; ++j) v_col[j] = 16 * g + 128 * j < c.D ? 16 * g + 128 * j : 0;
    }
    const int blk_shift = 31 - __clz(c.blk);
    uint32_t kr[2][KS], va[4][VW], vb[4][VW];
    float kscale = 0.f, vscale_a = 0.f, vscale_b = 0.f;
    // The tile to be loaded next: its first token, its place in its page, and
    // pointers that move along with it and start anew in every page.
    int t_load = t_begin + 16 * warp, page = t_load / c.P, row = t_load - page * c.P;
    bool mapped = false;
    const uint8_t *k_at = nullptr, *v_at = nullptr;
    const float *ks_at = nullptr, *vs_at = nullptr;
    auto enter_page = [&]() {
        mapped = false;
        if (t_load >= t_end) return;
        int phys = page;
        if (c.table) {
            phys = __ldg(c.table + static_cast<int64_t>(b) * c.pps + page);
            if (static_cast<unsigned>(phys) >= static_cast<unsigned>(c.num_pages)) {
                report(c.status, AKV_ERR_BAD_BLOCK_TABLE);
                return;
            }
        }
        mapped = true;
        k_at = c.k.codes + code_offset(c.k, b, h, phys, row) + g * c.k.sT;
        v_at = c.v.codes + code_offset(c.v, b, h, phys, row) + 2 * cc * c.v.sT;
        ks_at = c.k.scales + scale_offset(c.k, b, h, phys, 0);
        vs_at = c.v.scales + scale_offset(c.v, b, h, phys, 0);
    };
    const int64_t k_step = 16 * kStepWarps * c.k.sT, v_step = 16 * kStepWarps * c.v.sT;
    auto next_tile = [&]() {
        t_load += 16 * kStepWarps;
        row += 16 * kStepWarps;
        k_at += k_step;
        v_at += v_step;
        if (row >= c.P) {
            do {
                row -= c.P;
                ++page;
            } while (row >= c.P);
            enter_page();
        }
    };
    auto load_k = [&]() {
        const uint8_t* at8 = k_at + 8 * c.k.sT;
        auto load_rows = [&](auto in) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (in(i)) w = load_stream((i ? at8 : k_at) + k_col[j]);
                    kr[i][4 * j] = w.x; kr[i][4 * j + 1] = w.y; kr[i][4 * j + 2] = w.z; kr[i][4 * j + 3] = w.w;
                }
        };
        if (mapped && t_load + 16 <= t_end) {
            kscale = __ldg(ks_at + (row >> blk_shift));
            load_rows([](int) { return true; });
        } else {
            kscale = mapped && t_load < t_end ? __ldg(ks_at + (row >> blk_shift)) : 0.f;
            load_rows([&](int i) { return mapped && t_load + g + 8 * i < t_end; });
        }
    };
    auto load_v = [&](uint32_t (&vr)[4][VW], float& vscale) {
        auto load_rows = [&](auto in) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* at = v_at + (i & 1 ? c.v.sT : 0) + (i & 2 ? 8 * c.v.sT : 0);
                if (DP == 64) {
                    uint2 w = make_uint2(0, 0);
                    if (in(i)) w = load_stream8(at + v_col[0]);
                    vr[i][0] = w.x; vr[i][1] = w.y;
                } else {
#pragma unroll
                    for (int j = 0; j < DP / 128; ++j) {
                        uint4 w = make_uint4(0, 0, 0, 0);
                        if (in(i)) w = load_stream(at + v_col[j]);
                        vr[i][4 * j] = w.x; vr[i][4 * j + 1] = w.y; vr[i][4 * j + 2] = w.z; vr[i][4 * j + 3] = w.w;
                    }
                }
            }
        };
        if (mapped && t_load + 16 <= t_end) {
            vscale = __ldg(vs_at + (row >> blk_shift));
            load_rows([](int) { return true; });
        } else {
            vscale = mapped && t_load < t_end ? __ldg(vs_at + (row >> blk_shift)) : 0.f;
            load_rows([&](int i) { return mapped && t_load + 2 * cc + (i & 1) + 8 * (i >> 1) < t_end; });
        }
    };

    enter_page();
    load_k();
    load_v(va, vscale_a);

    // Query fragments: n = g, d as in load_k.
    float factor[NT][2];   // of the lane's score columns, rows 2c and 2c + 1
    int bound[NT][2];      // tokens that those rows see (rows past the last: all)
    int bound_min = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = TWIN ? g & 3 : 8 * nt + g;
        const bool in = r < rows;
        float x[DP / 64][16];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            if (in && 16 * cc + 64 * j < c.D) {
                load_q16(p, q_row(p, b, h, r0 + r) + 16 * cc + 64 * j, x[j]);
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k) x[j][k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) top = __uint_as_float(max(__float_as_uint(top), abs_bits(x[j][k])));
        }
        uint32_t tb = __float_as_uint(top);
        tb = max(tb, __shfl_xor_sync(0xFFFFFFFFu, tb, 1));
        tb = max(tb, __shfl_xor_sync(0xFFFFFFFFu, tb, 2));
        const int e = row_exponent(__uint_as_float(tb));
        const float up = power_of_two(e);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = x[s / 4][4 * (s % 4) + k] * up;
            const uint32_t h0 = pack_half2(y[0], y[1]), h1 = pack_half2(y[2], y[3]);
            if (warp == 0) {
                qs[s][nt][0][lane] = make_uint2(h0, h1);
                if (QLO) qs[s][nt][1][lane] = make_uint2(pack_rest(y[0], y[1], h0), pack_rest(y[2], y[3], h1));
            }
        }
        const float f = p.c2 * power_of_two(-e);
        const int bnd = in ? seen_by(p, (r0 + r) / p.G, len, qlen) : INT_MAX;
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
        for (int k = 0; k < 2; ++k) { base[nt][k] = 0.f; limit[nt][k] = -CUDART_INF_F; l[nt][k] = 0.f; if (PLO) carry[2 * nt + k][threadIdx.x] = 1.f; }
    }

    auto tile = [&](int t0, const uint32_t (&vr)[4][VW], float vscale, uint32_t (&v_next)[4][VW], float& vscale_next) {
        // Two sums per score: the tensor cores truncate as they add.
        float s[NT][4], s1[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[nt][k] = s1[nt][k] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t a0, a1, a2, a3;
            codes_to_half<FMT>(kr[0][k], a0, a2);
            codes_to_half<FMT>(kr[1][k], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float(&d)[4] = k & 1 ? s1[nt] : s[nt];
                const uint2 q = qs[k][nt][0][lane];
                mma16816(d, a0, a1, a2, a3, q.x, q.y);
                if (QLO) {
                    const uint2 ql = qs[k][nt][QLO ? 1 : 0][lane];
                    mma16816(d, a0, a1, a2, a3, ql.x, ql.y);
                }
            }
        }
        const float ks = kscale;
        // A NaN scale has to stay one: in lv, which makes the scores of what is
        // seen NaN; in iv it would reach the sums of rows that do not see it.
        const float vs = vscale < 8.0779357e-28f ? 8.0779357e-28f : vscale;
        const float lv = log2_fast(vs), iv = isnan(lv) ? 0.f : exp2_fast(-lv);
        next_tile();
        load_k();
        load_v(v_next, vscale_next);

        const bool all_seen = t0 + 16 <= bound_min;
        bool above = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float f[2] = {ks * factor[nt][0], ks * factor[nt][1]};
#pragma unroll
            for (int k = 0; k < 4; ++k) s[nt][k] += s1[nt][k];
            if (p.scores) {
                float* to = p.scores + (static_cast<int64_t>(bh) * c.T + t0 + g) * p.R + r0 + 8 * nt + 2 * cc;
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    if (t0 + g + 4 * k >= t_end || 8 * nt + 2 * cc >= rows) continue;
                    if (p.R % 2 == 0) {
                        *reinterpret_cast<float2*>(to + k * 4 * p.R) = make_float2(s[nt][k] * f[0], s[nt][k + 1] * f[1]);
                    } else {
                        to[k * 4 * p.R] = s[nt][k] * f[0];
                        if (8 * nt + 2 * cc + 1 < rows) to[k * 4 * p.R + 1] = s[nt][k + 1] * f[1];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s[nt][k] = fmaf(s[nt][k], f[k & 1], lv);
                if (!all_seen && t0 + g + 8 * (k >> 1) >= bound[nt][k & 1]) s[nt][k] = -CUDART_INF_F;
                above |= s[nt][k] > limit[nt][k & 1];
            }
        }
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
                    const float alpha = limit[nt][k] == -CUDART_INF_F ? 0.f : exp2_fast(base[nt][k] - to);
                    base[nt][k] = to;
                    limit[nt][k] = up ? __fadd_rd(to, 15.5f) : limit[nt][k];
                    l[nt][k] *= alpha;
                    if (PLO) carry[2 * nt + k][threadIdx.x] *= alpha;
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
                s[nt][k] = exp2_fast(s[nt][k] - base[nt][k & 1]);
                l[nt][k & 1] = fmaf(s[nt][k], iv, l[nt][k & 1]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t hi = pack_half2(s[nt][2 * k], s[nt][2 * k + 1]);
                if (SECOND) pl[nt][k] = transpose8x8(pack_rest(s[nt][2 * k], s[nt][2 * k + 1], hi));
                if (TWIN && cc >= 2) hi = pack_rest(s[nt][2 * k], s[nt][2 * k + 1], hi);
                ph[nt][k] = transpose8x8(hi);
            }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            // Bytes of tokens (0, 1) and (2, 3) of the lane side by side: four d, two d-tiles.
            const uint32_t e0 = __byte_perm(vr[0][w], vr[1][w], 0x5140), e1 = __byte_perm(vr[0][w], vr[1][w], 0x7362);
            const uint32_t f0 = __byte_perm(vr[2][w], vr[3][w], 0x5140), f1 = __byte_perm(vr[2][w], vr[3][w], 0x7362);
            uint32_t a[2][4];
            codes_to_half<FMT>(e0, a[0][0], a[0][1]);
            codes_to_half<FMT>(f0, a[0][2], a[0][3]);
            codes_to_half<FMT>(e1, a[1][0], a[1][1]);
            codes_to_half<FMT>(f1, a[1][2], a[1][3]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816(o[2 * w + j][nt], a[j][0], a[j][1], a[j][2], a[j][3], ph[nt][0], ph[nt][1]);
                    if (SECOND) mma16816(o[2 * w + j][nt], a[j][0], a[j][1], a[j][2], a[j][3], pl[SECOND ? nt : 0][0], pl[SECOND ? nt : 0][1]);
                }
        }
    };
    // O's sum, brought to the present base by `carry`: the lane's own part of
    // the room that `red` takes at the end.
    float4* const sums = reinterpret_cast<float4*>(&red[warp][0][0]) + lane;
    for (int t0 = t_begin + 16 * warp; t0 < t_end; t0 += 32 * kStepWarps) {
        tile(t0, va, vscale_a, vb, vscale_b);
        if (t0 + 16 * kStepWarps < t_end) tile(t0 + 16 * kStepWarps, vb, vscale_b, va, vscale_a);
        if (PLO && t0 % FOLD >= FOLD - 32 * kStepWarps) {
            const bool first = t0 - t_begin < FOLD;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float f0 = carry[2 * nt][threadIdx.x], f1 = carry[2 * nt + 1][threadIdx.x];
                carry[2 * nt][threadIdx.x] = carry[2 * nt + 1][threadIdx.x] = 1.f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    float(&x)[4] = o[i][nt];
                    float4 v = first ? make_float4(0.f, 0.f, 0.f, 0.f) : sums[(i * NT + nt) * 32];
                    v = make_float4(fmaf(v.x, f0, x[0]), fmaf(v.y, f1, x[1]), fmaf(v.z, f0, x[2]), fmaf(v.w, f1, x[3]));
                    sums[(i * NT + nt) * 32] = v;
                    x[0] = x[1] = x[2] = x[3] = 0.f;
                }
            }
        }
    }

    allow_next_kernel();
    const int begun = t_begin + 16 * warp;
    if (PLO && begun + (FOLD - 1 - begun % FOLD) / (32 * kStepWarps) * (32 * kStepWarps) < t_end) {  // there is a sum
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
            for (int i = 0; i < KS; ++i) {
                // Byte x of the lane group's bytes.
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int x = 2 * i + j;
                    const int d = DP == 64 ? 8 * g + x : 128 * (x / 16) + 16 * g + x % 16;
                    red[warp][r][d] = o[i][nt][k + 2 * j] * a;
                }
            }
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
        } else {
            const int64_t row = out_row(p, b, h, r0 + r);
            const float lse = none ? -CUDART_INF_F : top + log2f(sum);
            if (p.lse) p.lse[row] = lse;
            if (p.lse_out) p.lse_out[row] = lse * 0.69314718055994531f;
        }
    }
    __syncthreads();
    // Four dimensions a thread, so many rows at a time.
    const int lanes = c.D / 4, row_step = kStepThreads / lanes, d = threadIdx.x % lanes * 4;
    for (int r = threadIdx.x / lanes; r < rows && threadIdx.x < lanes * row_step; r += row_step) {
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
            store4(p.out, p.out_dtype, out_row(p, b, h, r0 + r) * c.D + d, f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
        }
    }
    if constexpr (CLUSTER) {
        __syncthreads();
        cluster_sync();
        // Row r is finished by CTA r % ranks, its pieces in the order of the CTAs.
        for (int r = rank; r < rows; r += ranks) {
            float top = -CUDART_INF_F, sum = 0.f;
            float2 v[kStepCluster];
#pragma unroll
            for (int k = 0; k < kStepCluster; ++k) {
                v[k] = k < ranks ? load_remote2(&piece[r], k) : make_float2(-CUDART_INF_F, 0.f);
                top = fmaxf(top, v[k].x);
            }
#pragma unroll
            for (int k = 0; k < kStepCluster; ++k)
                if (v[k].x != -CUDART_INF_F) sum += v[k].y * exp2f(v[k].x - top);
            const bool none = top == -CUDART_INF_F && !isnan(sum);
            const int64_t row = out_row(p, b, h, r0 + r);
            if (static_cast<int>(threadIdx.x) < lanes) {
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < kStepCluster; ++k) {
                    if (v[k].x == -CUDART_INF_F) continue;
                    const float f = exp2f(v[k].x - top);
                    const float4 o = load_remote4(&red[0][r][d], k);
                    acc.x = fmaf(o.x, f, acc.x); acc.y = fmaf(o.y, f, acc.y);
                    acc.z = fmaf(o.z, f, acc.z); acc.w = fmaf(o.w, f, acc.w);
                }
                const float f = none ? 0.f : 1.f / sum;
                store4(p.out, p.out_dtype, row * c.D + d, none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
            }
            if (threadIdx.x == 0) {
                const float lse = none ? -CUDART_INF_F : isnan(sum) ? sum : top + log2f(sum);
                if (p.lse) p.lse[row] = lse;
                if (p.lse_out) p.lse_out[row] = lse * 0.69314718055994531f;
            }
        }
        __syncthreads();
        cluster_sync();  // nobody reads this CTA's memory any more
        return;
    }
    // On to the next unit.
    at += n_mine;
    chunk = 0;
    if (++unit_of_b == units) {
        unit_of_b = 0;
        do ++b;
        while (b < c.B && share_chunks(p, b) == 0);
    }
    __syncthreads();
    }
}

}  // namespace q8
}  // namespace akv
