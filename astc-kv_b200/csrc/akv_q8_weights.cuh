// Accumulated token weights where the rows (query tokens x heads of a kv
// head) are too many to keep their scores: the scores are computed again
// from K and the finished log-sum-exp, sum over rows of 2^(s - lse).
//
// A warp keeps 32 tokens' K as tensor-core fragments in registers and goes
// through the rows, eight at a time, which the CTA brings to shared memory
// as fragments (S^T = K Q^T as in the step kernel). A token's weight is
// summed by one warp in the order of the rows, so it does not depend on
// timing. Half the products of the attention itself, and one exp2 a score.
#pragma once
#include "akv_q8_attend.cuh"

namespace akv {
namespace q8 {

constexpr int kWeightWarps = 4;
constexpr int kWeightThreads = 32 * kWeightWarps;
constexpr int kWeightTile = 32 * kWeightWarps;  // tokens per CTA
constexpr int kWeightRows = 32;                 // rows in shared memory at a time

template <int FMT, int DP, bool QLO>
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(AttnParams p) {
    constexpr int KS = DP / 16;
    __shared__ uint2 qs[kWeightRows / 8][KS][QLO ? 2 : 1][32];
    __shared__ float3 info[kWeightRows];  // factor, lse, tokens seen

    const CacheDev& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z, bh = b * c.H + h;
    const int len = len_of(p, b), qlen = q_len_of(p, b);
    const int first = blockIdx.x * kWeightTile;
    float* at = p.weights + static_cast<int64_t>(bh) * p.wstride;
    if (first >= len) {
        if (!p.accumulate && first + threadIdx.x < c.T) at[first + threadIdx.x] = 0.f;
        return;
    }
    const int t0 = first + 32 * warp;

    uint32_t a[2][KS][4];
    float ks[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int tt = t0 + 16 * i;
        int row = 0;
        const int phys = tt < len ? page_of(c, b, tt, row) : -1;
        const uint8_t* base = c.k.codes + b * c.k.sB + h * c.k.sH + phys * c.k.sP + row * c.k.sT;
        ks[i] = phys >= 0 ? c.k.scales[b * c.k.cB + h * c.k.cH + phys * c.k.cP + row / c.blk] : 0.f;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            uint4 w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                w[k] = make_uint4(0, 0, 0, 0);
                if (phys >= 0 && tt + g + 8 * k < len && 16 * cc + 64 * j < c.D)
                    w[k] = load_stream(base + (g + 8 * k) * c.k.sT + 16 * cc + 64 * j);
            }
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

    // The first query that sees the CTA's first token; rows end with the queries.
    const int i0 = p.causal ? max(first - (len - qlen), 0) : 0;
    const int r_end = qlen * p.G;
    float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    for (int r0 = i0 * p.G; r0 < r_end; r0 += kWeightRows) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kWeightRows / 8 / kWeightWarps; ++q) {
            const int grp = warp + q * kWeightWarps, r = r0 + 8 * grp + g;
            float x[DP / 64][16];
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) {
                if (r < r_end && 16 * cc + 64 * j < c.D) {
                    load_q16(p, q_row(p, b, h, r) + 16 * cc + 64 * j, x[j]);
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
                qs[grp][s][0][lane] = make_uint2(h0, h1);
                if (QLO) qs[grp][s][QLO ? 1 : 0][lane] = make_uint2(pack_rest(y[0], y[1], h0), pack_rest(y[2], y[3], h1));
            }
            if (cc == 0) {
                const int seen = r < r_end ? seen_by(p, r / p.G, len, qlen) : 0;
                info[8 * grp + g] = make_float3(p.c2 * power_of_two(-e), seen ? p.lse[out_row(p, b, h, r)] : 0.f, __int_as_float(seen));
            }
        }
        __syncthreads();
#pragma unroll
        for (int grp = 0; grp < kWeightRows / 8; ++grp) {
            if (r0 + 8 * grp >= r_end) break;
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
#pragma unroll
                for (int q = 0; q < (QLO ? 2 : 1); ++q) {
                    const uint2 f = qs[grp][k][q][lane];
#pragma unroll
                    for (int i = 0; i < 2; ++i) mma16816(s[i], a[i][k][0], a[i][k][1], a[i][k][2], a[i][k][3], f.x, f.y);
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float3 f = info[8 * grp + 2 * cc + k];
                const int seen = __float_as_int(f.z);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (t0 + 16 * i + g + 8 * j < seen) sum[i][j] += exp2_fast(s[i][2 * j + k] * (ks[i] * f.x) - f.y);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float w = sum[i][j];
            w += __shfl_xor_sync(0xFFFFFFFFu, w, 1);
            w += __shfl_xor_sync(0xFFFFFFFFu, w, 2);
            const int t = t0 + 16 * i + g + 8 * j;
            if (cc == 0 && t < c.T) {
                if (!p.accumulate) at[t] = t < len ? w : 0.f;
                else if (t < len) at[t] += w;
            }
        }
}

}  // namespace q8
}  // namespace akv
