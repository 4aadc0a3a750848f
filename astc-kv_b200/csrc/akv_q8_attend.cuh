// Attention over the 8-bit KV cache: parameters and helpers shared by the
// kernels, the split combine, and the accumulated token weights.
#pragma once
#include <math_constants.h>

#include "akv_q8_common.cuh"

namespace akv {
namespace q8 {

struct AttnParams {
    CacheDev c;
    int Hq, G, n;               // query heads, per kv head, query tokens
    int R;                      // rows of a kv head: n * G, row r = query token r / G, head r % G
    int q_dtype, out_dtype, causal, accumulate;
    int q_vec;                  // query rows start on 16-byte boundaries
    float c2;                   // scale * log2(e)
    const void* q;
    int64_t qB, qT, qH;         // elements
    const int32_t* lens;
    const int32_t* q_lens;
    int split, nsplits;         // tokens per split
    float* part_o;              // [B][H][nsplits][R][D]
    float2* part_ml;            // [B][H][nsplits][R]
    float* scores;              // [B][H][T][R], base 2, or NULL
    void* out;
    float* lse;                 // [B][n][Hq], base 2, or NULL
    float* lse_out;             // [B][n][Hq], natural, or NULL
    float* weights;
    int64_t wstride;
};

__device__ __forceinline__ int len_of(const AttnParams& p, int b) { return p.lens ? min(max(p.lens[b], 0), p.c.T) : p.c.T; }
__device__ __forceinline__ int q_len_of(const AttnParams& p, int b) { return p.q_lens ? min(max(p.q_lens[b], 0), p.n) : p.n; }
// Tokens that query i of a sequence sees.
__device__ __forceinline__ int seen_by(const AttnParams& p, int i, int len, int qlen) {
    if (i >= qlen) return 0;
    return p.causal ? max(len - qlen + i + 1, 0) : len;
}
__device__ __forceinline__ int64_t q_row(const AttnParams& p, int b, int h, int r) {
    return b * p.qB + (r / p.G) * p.qT + (h * p.G + r % p.G) * p.qH;
}
// Row r's place among [B][n][Hq].
__device__ __forceinline__ int64_t out_row(const AttnParams& p, int b, int h, int r) {
    return (static_cast<int64_t>(b) * p.n + r / p.G) * p.Hq + h * p.G + r % p.G;
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

// 16 consecutive query elements as floats.
__device__ __forceinline__ void load_q16(const AttnParams& p, int64_t at, float (&x)[16]) {
    if (!p.q_vec) {
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = load_elem(p.q, p.q_dtype, at + k);
    } else if (p.q_dtype == AKV_Q_F32) {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 v = __ldg(s + k);
            x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
        }
    } else {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint4 v = __ldg(s + k);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 f;
                if (p.q_dtype == AKV_Q_BF16) f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
                else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                x[8 * k + 2 * j] = f.x;
                x[8 * k + 2 * j + 1] = f.y;
            }
        }
    }
}

// The power of two that brings a query row's largest |x| to [2^14, 2^15), so
// that fp16 holds the row: bf16 and fp16 rows exactly, down to 2^-38 of the
// largest; fp32 rows in two parts. Rows of zeros, infinities or NaN stay.
__device__ __forceinline__ int row_exponent(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    if (top == 0.f || e == 128) return 0;
    return min(max(14 - e, -126), 126);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What fp16 rounding left of (a, b).
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack_half2(a - f.x, b - f.y);
}

// Four codes as two fp16 pairs, exactly. int8: code + 128 becomes the low
// byte of 1024 + (code + 128), and 1152 is taken off. e4m3: the conversion
// instruction.
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FMT == AKV_Q8_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const uint32_t c = 0x64806480u;
        const __half2 base = *reinterpret_cast<const __half2*>(&c);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), base), y = __hsub2(*reinterpret_cast<const __half2*>(&b), base);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}\n" : "=r"(lo), "=r"(hi) : "r"(w));
    }
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transposes an 8x8 matrix of 16-bit elements spread over the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load_stream8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// ------------------------------------------------------------------ combine

constexpr int kCombineThreads = 128;
constexpr int kWeightTokens = 512;   // per CTA of the weights part

// Base-2 log-sum-exp of row r over the splits, by one warp; all lanes get it.
__device__ __forceinline__ float combined_lse(const float2* ml, int nsplits, int R) {
    const int lane = threadIdx.x & 31;
    float m = -CUDART_INF_F;
    for (int s = lane; s < nsplits; s += 32) m = fmaxf(m, ml[static_cast<int64_t>(s) * R].x);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    float l = 0.f;
    for (int s = lane; s < nsplits; s += 32) {
        const float2 v = ml[static_cast<int64_t>(s) * R];
        if (v.x != -CUDART_INF_F) l += v.y * exp2f(v.x - m);
    }
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    return isnan(l) ? l : m == -CUDART_INF_F ? m : m + log2f(l);
}

// Blocks [0, rows): one row of the output each: the splits' partials weighted
// by 2^(m - lse), added in the order of the splits. Blocks from `rows` on:
// 512 tokens of one kv head each: the stored scores of its rows become
// softmax weights, which are added up.
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(AttnParams p, int rows, int wblocks) {
    __shared__ float lse[16];
    __shared__ int ends[16];
    const int tid = threadIdx.x;
    if (static_cast<int>(blockIdx.x) < rows) {
        const int r = blockIdx.x % p.R, bh = blockIdx.x / p.R, h = bh % p.c.H, b = bh / p.c.H;
        const float2* ml = p.part_ml + static_cast<int64_t>(bh) * p.nsplits * p.R + r;
        const float all = combined_lse(ml, p.nsplits, p.R);
        const int64_t row = out_row(p, b, h, r);
        if (tid == 0) {
            if (p.lse) p.lse[row] = all;
            if (p.lse_out) p.lse_out[row] = all * 0.69314718055994531f;
        }
        const float* o = p.part_o + (static_cast<int64_t>(bh) * p.nsplits * p.R + r) * p.c.D;
        const int64_t step = static_cast<int64_t>(p.R) * p.c.D;
        for (int d = tid; d < p.c.D; d += kCombineThreads) {
            float a = 0.f;
            for (int s0 = 0; s0 < p.nsplits; s0 += 8) {
                float x[8], w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int s = s0 + k;
                    w[k] = s < p.nsplits ? ml[static_cast<int64_t>(s) * p.R].x : -CUDART_INF_F;
                    x[k] = w[k] != -CUDART_INF_F ? o[s * step + d] : 0.f;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (w[k] != -CUDART_INF_F) a = fmaf(x[k], exp2f(w[k] - all), a);
            }
            store_elem(p.out, p.out_dtype, row * p.c.D + d, a);
        }
        return;
    }
    const int wb = blockIdx.x - rows, bh = wb / wblocks, h = bh % p.c.H, b = bh / p.c.H, t0 = wb % wblocks * kWeightTokens;
    const int len = len_of(p, b), qlen = q_len_of(p, b);
    if (p.accumulate && t0 >= len) return;
    for (int r = tid >> 5; r < p.R; r += kCombineThreads / 32) {
        const float v = combined_lse(p.part_ml + static_cast<int64_t>(bh) * p.nsplits * p.R + r, p.nsplits, p.R);
        if ((tid & 31) == 0) {
            lse[r] = v;
            ends[r] = seen_by(p, r / p.G, len, qlen);
        }
    }
    __syncthreads();
    const float* sc = p.scores + static_cast<int64_t>(bh) * p.c.T * p.R;
    float* at = p.weights + static_cast<int64_t>(bh) * p.wstride;
    for (int t = t0 + tid; t < min(t0 + kWeightTokens, p.c.T); t += kCombineThreads) {
        float w = 0.f;
        for (int r = 0; r < p.R; ++r)
            if (t < ends[r]) w += exp2f(sc[static_cast<int64_t>(t) * p.R + r] - lse[r]);
        if (!p.accumulate) at[t] = w;
        else if (t < len) at[t] += w;
    }
}

}  // namespace q8
}  // namespace akv
