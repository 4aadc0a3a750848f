// Accumulated token weights where the rows (query tokens x heads of a kv
// head) are too many to keep their scores: the scores are computed again
// from K and the finished log-sum-exp, sum over rows of 2^(s - lse).
//
// The query rows are laid out once as tensor-core fragments (by blocks of the
// combine launch, pack_rows). A warp keeps 32 tokens' K as fragments in
// registers and goes through the rows, eight at a time (S^T = K Q^T as in the
// step kernel); the CTA's eight warps are four groups of 32 tokens times two
// halves of the rows, and the rows' fragments come to shared memory by
// asynchronous copies one stage ahead. A token's two sums are added in a fixed
// order, so the result does not depend on timing.
//
// A score is one chain of products here and two in the step kernel, so it may
// differ in its last bits from the one that went into the log-sum-exp; measured
// against 64 bits, weights of 40 to 1200 rows are 1e-7 to 6e-7 off, those of
// plain fp32 1e-7 to 9e-7.
//
// Half the products of the attention itself and one exp2 a score, of which an
// SM does 16 a cycle: 90 us for 3 x 452 query tokens against 18578, 16/16
// heads, D 64, where it takes 274 us.
#pragma once
#include "akv_q8_attend.cuh"

namespace akv {
namespace q8 {

constexpr int kWeightThreads = 256;
constexpr int kWeightTile = 128;  // tokens per CTA

// Row groups of a stage: 16 KB of fragments.
template <int DP, bool QLO>
constexpr int kWeightGroups = 64 / (DP / 16 * (QLO ? 2 : 1));

__device__ __forceinline__ void copy_async16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int FMT, int DP, bool QLO>
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(AttnParams p) {
    constexpr int KS = DP / 16, GROUPS = kWeightGroups<DP, QLO>, PARTS = QLO ? 2 : 1;
    __shared__ __align__(16) uint2 qs[2][GROUPS][KS][PARTS][32];
    __shared__ float2 info[2][GROUPS * 8];  // factor, lse
    __shared__ float half_sum[kWeightTile];

    const CacheDev& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z, bh = b * c.H + h;
    const int len = len_of(p, b), qlen = q_len_of(p, b);
    const int first = blockIdx.x * kWeightTile;
    float* at = p.weights + static_cast<int64_t>(bh) * p.wstride;
    if (first >= len) {
        // So that the kernel does not end before the one before it.
        if (blockIdx.x == 0) wait_for_previous_kernel();
        if (!p.accumulate && threadIdx.x < kWeightTile && first + threadIdx.x < c.T) at[first + threadIdx.x] = 0.f;
        return;
    }
    const int t0 = first + 32 * (warp & 3);

    uint32_t a[2][KS][4];
    float ks[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int tt = t0 + 16 * i;
        int row = 0;
        const int phys = tt < len ? page_of(c, b, tt, row) : -1;
        const uint8_t* base = c.k.codes + b * c.k.sB + h * c.k.sH + phys * c.k.sP + row * c.k.sT;
        ks[i] = phys >= 0 ? c.k.scales[scale_offset(c.k, b, h, phys, row / c.blk)] : 0.f;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            uint4 w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                w[k] = load_stream_if(base + (g + 8 * k) * c.k.sT + 16 * cc + 64 * j,
                                      phys >= 0 && tt + g + 8 * k < len && 16 * cc + 64 * j < c.D);
            codes_to_half<FMT>(w[0].x, a[i][4 * j][0], a[i][4 * j][2]);
            codes_to_half<FMT>(w[1].x, a[i][4 * j][1], a[i][4 * j][3]);
            codes_to_half<FMT>(w[0].y, a[i][4 * j + 1][0], a[i][4 * j + 1][2]);
            codes_to_half<FMT>(w[1].y, a[i][4 * j + 1][1], a[i][4 * j + 1][3]);
            codes_to_half<FMT>(w[0].z, a[i][4 * j + 2][0], a[i][4 * j + 2][2]);
            codes_to_half<FMT>(w[1].z, a[i][4 * j + 2][1], a[i][4 * j + 2][3]);
            codes_to_half<FMT>(w[0].w, a[i][4 * j + 3][0], a[i][4 * j + 3][2]);
            codes_to_half<FMT>(w[1].w, a[i][4 * j + 3][1], a[i][4 * j + 3][3]);
        }
    }

    // Rows from the group of the first query that sees the CTA's first token
    // to the last query's.
    const int groups = (p.R + 7) / 8, r_end = qlen * p.G;
    const int g_first = p.causal ? max(first - (len - qlen), 0) * p.G / 8 : 0, g_end = (r_end + 7) / 8;
    // Rows from here on see the whole tile. (A row that sees nothing has lse
    // -inf, which the mask keeps out.)
    const int r_full = max(p.causal ? first + kWeightTile - 1 - (len - qlen) : (len >= first + kWeightTile ? 0 : qlen), 0) * p.G;
    const uint2* q = p.q_rows + static_cast<int64_t>(bh) * groups * KS * PARTS * 32;
    const float* factors = p.q_factors + static_cast<int64_t>(bh) * groups * 8;
    wait_for_previous_kernel();
    auto fetch = [&](int g0, int stage) {
        const int n = min(GROUPS, g_end - g0) * KS * PARTS * 16;  // 16-byte pieces
        const uint4* from = reinterpret_cast<const uint4*>(q + static_cast<int64_t>(g0) * KS * PARTS * 32);
        uint4* to = reinterpret_cast<uint4*>(qs[stage]);
        for (int i = threadIdx.x; i < n; i += kWeightThreads) copy_async16(to + i, from + i);
        copy_commit();
        for (int i = threadIdx.x; i < GROUPS * 8; i += kWeightThreads) {
            const int r = 8 * g0 + i;
            info[stage][i] = r < r_end ? make_float2(factors[r], p.lse[out_row(p, b, h, r)]) : make_float2(0.f, CUDART_INF_F);
        }
    };
    float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    if (g_first < g_end) fetch(g_first, 0);
    for (int g0 = g_first, stage = 0; g0 < g_end; g0 += GROUPS, stage ^= 1) {
        if (g0 + GROUPS < g_end) {
            fetch(g0 + GROUPS, stage ^ 1);
            copy_wait<1>();
        } else {
            copy_wait<0>();
        }
        __syncthreads();
        for (int grp = warp >> 2; grp < GROUPS && g0 + grp < g_end; grp += 2) {
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const uint2 f = qs[stage][grp][k][part][lane];
#pragma unroll
                    for (int i = 0; i < 2; ++i) mma16816(s[i], a[i][k][0], a[i][k][1], a[i][k][2], a[i][k][3], f.x, f.y);
                }
            }
            const int r0 = 8 * (g0 + grp);
            const bool all_seen = r0 >= r_full && r0 + 8 <= r_end;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 f = info[stage][8 * grp + 2 * cc + k];
                const float f0 = ks[0] * f.x, f1 = ks[1] * f.x;
                float e[2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    e[0][j] = exp2_fast(fmaf(s[0][2 * j + k], f0, -f.y));
                    e[1][j] = exp2_fast(fmaf(s[1][2 * j + k], f1, -f.y));
                }
                if (!all_seen) {
                    const int r = r0 + 2 * cc + k, seen = r < r_end ? seen_by(p, r / p.G, len, qlen) : 0;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            if (t0 + 16 * i + g + 8 * j >= seen) e[i][j] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) sum[i][j] += e[i][j];
            }
        }
        __syncthreads();  // the stage may be filled again
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            sum[i][j] += __shfl_xor_sync(0xFFFFFFFFu, sum[i][j], 1);
            sum[i][j] += __shfl_xor_sync(0xFFFFFFFFu, sum[i][j], 2);
            if (warp >= 4 && cc == 0) half_sum[32 * (warp & 3) + 16 * i + g + 8 * j] = sum[i][j];
        }
    __syncthreads();
    if (warp >= 4 || cc != 0) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int t = t0 + 16 * i + g + 8 * j;
            if (t >= c.T) continue;
            const float w = sum[i][j] + half_sum[t - first];
            if (!p.accumulate) at[t] = t < len ? w : 0.f;
            else if (t < len) at[t] += w;
        }
}

}  // namespace q8
}  // namespace akv
