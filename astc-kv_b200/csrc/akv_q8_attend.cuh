// Attention over the 8-bit KV cache.
#pragma once
#include <math_constants.h>

#include "akv_q8_common.cuh"

namespace akv {
namespace q8 {

struct AttnParams {
    CacheDev c;
    int Hq, G, n;               // query heads, per kv head, query tokens
    int q_dtype, out_dtype, causal, accumulate;
    float c2;                   // scale * log2(e)
    const void* q;
    int64_t qB, qT, qH;
    const int32_t* lens;
    const int32_t* q_lens;
    void* out;
    float* lse;                 // base 2, workspace
    float* lse_out;
    float* weights;
    int64_t wstride;
};

__device__ __forceinline__ int len_of(const AttnParams& p, int b) {
    return p.lens ? min(max(p.lens[b], 0), p.c.T) : p.c.T;
}
__device__ __forceinline__ int q_len_of(const AttnParams& p, int b) {
    return p.q_lens ? min(max(p.q_lens[b], 0), p.n) : p.n;
}
// Tokens that query i of sequence b sees.
__device__ __forceinline__ int seen_by(const AttnParams& p, int i, int len, int qlen) {
    if (i >= qlen) return 0;
    return p.causal ? max(len - qlen + i + 1, 0) : len;
}
__device__ __forceinline__ float load_elem(const void* q, int dtype, int64_t i) {
    if (dtype == AKV_Q_F32) return static_cast<const float*>(q)[i];
    if (dtype == AKV_Q_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(q)[i]);
    return __half2float(static_cast<const __half*>(q)[i]);
}
__device__ __forceinline__ void store_elem(void* o, int dtype, int64_t i, float v) {
    if (dtype == AKV_Q_F32) static_cast<float*>(o)[i] = v;
    else if (dtype == AKV_Q_BF16) static_cast<__nv_bfloat16*>(o)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(o)[i] = __float2half_rn(v);
}

constexpr int kRowThreads = 128;

// q . K[t] of one token, q in shared memory.
template <int FMT>
__device__ __forceinline__ float score(const AttnParams& p, const float* q, int b, int h, int t) {
    const SideDev& s = p.c.k;
    const int phys = page_of(p.c, b, t), row = t % p.c.P;
    if (phys < 0) return 0.f;
    const uint8_t* k = s.codes + code_offset(s, b, h, phys, row);
    float a = 0.f;
    for (int d = 0; d < p.c.D; ++d) a = fmaf(q[d], from_code<FMT>(k[d]), a);
    return a * s.scales[scale_offset(s, b, h, phys, row / p.c.blk)] * p.c2;
}

// One CTA per (query head, query token, sequence): 128 tokens at a time with
// a running maximum and sum.
template <int FMT>
__global__ void __launch_bounds__(kRowThreads) attend_kernel(AttnParams p) {
    __shared__ float q[256], pr[kRowThreads], red[4];
    const int hq = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, h = hq / p.G, D = p.c.D;
    const int end = seen_by(p, i, len_of(p, b), q_len_of(p, b));
    for (int d = tid; d < D; d += kRowThreads) q[d] = load_elem(p.q, p.q_dtype, b * p.qB + i * p.qT + hq * p.qH + d);
    __syncthreads();
    float m = -CUDART_INF_F, l = 0.f, o[2] = {0.f, 0.f};
    for (int t0 = 0; t0 < end; t0 += kRowThreads) {
        const int t = t0 + tid, n = min(kRowThreads, end - t0);
        const float s = t < end ? score<FMT>(p, q, b, h, t) : -CUDART_INF_F;
        float x = s;
        for (int k = 16; k; k >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, k));
        if (tid % 32 == 0) red[tid / 32] = x;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = mn == -CUDART_INF_F ? 0.f : mn, alpha = exp2f(m - base);
        const float e = t < end ? exp2f(s - base) : 0.f;
        pr[tid] = e;
        __syncthreads();
        float sum = 0.f;
        for (int k = 0; k < n; ++k) sum += pr[k];
        l = l * alpha + sum;
        m = mn;
        for (int j = 0; j < 2; ++j) {
            const int d = tid + j * kRowThreads;
            if (d >= D) continue;
            float a = 0.f;
            for (int k = 0; k < n; ++k) {
                const SideDev& v = p.c.v;
                const int phys = page_of(p.c, b, t0 + k), row = (t0 + k) % p.c.P;
                if (phys < 0) continue;
                a = fmaf(pr[k] * v.scales[scale_offset(v, b, h, phys, row / p.c.blk)],
                         from_code<FMT>(v.codes[code_offset(v, b, h, phys, row) + d]), a);
            }
            o[j] = o[j] * alpha + a;
        }
        __syncthreads();
    }
    const int64_t row = (static_cast<int64_t>(b) * p.n + i) * p.Hq + hq;
    for (int j = 0; j < 2; ++j)
        if (tid + j * kRowThreads < D) store_elem(p.out, p.out_dtype, row * D + tid + j * kRowThreads, end ? o[j] / l : 0.f);
    if (tid == 0) {
        const float lse = end ? m + log2f(l) : -CUDART_INF_F;
        p.lse[row] = lse;
        if (p.lse_out) p.lse_out[row] = lse * 0.69314718055994531f;
    }
}

// One CTA per (128 tokens, kv head, sequence).
template <int FMT>
__global__ void __launch_bounds__(kRowThreads) weights_kernel(AttnParams p) {
    __shared__ float q[256];
    const int h = blockIdx.y, b = blockIdx.z, t = blockIdx.x * kRowThreads + threadIdx.x;
    const int len = len_of(p, b), qlen = q_len_of(p, b);
    float w = 0.f;
    for (int r = 0; r < qlen * p.G; ++r) {
        const int i = r / p.G, hq = h * p.G + r % p.G;
        __syncthreads();
        for (int d = threadIdx.x; d < p.c.D; d += kRowThreads) q[d] = load_elem(p.q, p.q_dtype, b * p.qB + i * p.qT + hq * p.qH + d);
        __syncthreads();
        if (t < seen_by(p, i, len, qlen)) w += exp2f(score<FMT>(p, q, b, h, t) - p.lse[(static_cast<int64_t>(b) * p.n + i) * p.Hq + hq]);
    }
    if (t >= p.c.T) return;
    float* at = p.weights + (static_cast<int64_t>(b) * p.c.H + h) * p.wstride + t;
    if (p.accumulate) {
        if (t < len) *at += w;
    } else {
        *at = w;
    }
}

}  // namespace q8
}  // namespace akv
