// Attention over the 8-bit KV cache: parameters and helpers shared by the
// kernels, the split combine, and the accumulated token weights.
#pragma once
#include <climits>

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
    // Partials: of the chunk kernel [B][H][nsplits][R] rows, of the step
    // kernel two pieces for each CTA, row_group rows each (see Parts).
    int split, nsplits;         // tokens per split
    int share_ctas;             // CTAs of the step kernel, 0 for the chunk kernel, minus the size of its clusters
    int share_min;              // chunks that a share has at least
    int row_group;
    bool long_sums;             // of a CTA of the step kernel with a 16-bit output, see kStepLong
    float* part_o;              // ... [D], weighted by 2^-base
    float2* part_ml;            // base (-inf: nothing seen), sum
    uint2* q_rows;              // query rows as fragments for the weights kernel, see pack_rows
    float* q_factors;
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

__device__ __forceinline__ void store4(void* o, int dtype, int64_t i, float4 v) {
    if (dtype == AKV_Q_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(o) + i) = v;
    } else if (dtype == AKV_Q_BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(o) + i) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(static_cast<__half*>(o) + i) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
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
// that fp16 holds the row: bf16 elements exactly down to 2^-31 of the largest,
// below that off by 2^-39 of it at most; fp16 elements exactly, but for the
// last bit of subnormal ones in rows that reach 2^15; fp32 rows in two parts
// (22 bits). Rows of zeros, infinities or NaN stay.
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

__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// The same, or zeros without a load; nothing waits for what is loaded.
__device__ __forceinline__ uint4 load_stream_if(const void* p, bool in) {
    uint4 v;
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %5, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
        "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n}\n"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"(static_cast<uint32_t>(in)));
    return v;
}
__device__ __forceinline__ uint2 load_stream8_if(const void* p, bool in) {
    uint2 v;
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %3, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\n"
        "@p ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n}\n"
        : "=&r"(v.x), "=&r"(v.y) : "l"(p), "r"(static_cast<uint32_t>(in)));
    return v;
}

// ------------------------------------------------------------------ combine

constexpr int kCombineThreads = 256;

// ------------------------------------------------- the step kernel's shares

constexpr int kShareTokens = 64;

// 64-token chunks of each (kv head, row group) of sequence b.
__device__ __forceinline__ int share_chunks(const AttnParams& p, int b) {
    return q_len_of(p, b) > 0 ? (len_of(p, b) + kShareTokens - 1) / kShareTokens : 0;
}

// a / b of numbers that are not negative; most fit 32 bits, whose division is
// several times shorter.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// CTA i does chunks [start(i), start(i + 1)) of all, counted by sequence, kv
// head and row group, and along the tokens.
struct Shares {
    int64_t chunks;
    int ctas;
    __device__ __forceinline__ int64_t start(int i) const { return quotient(i * chunks, ctas); }
    __device__ __forceinline__ int owner(int64_t chunk) const { return static_cast<int>(quotient((chunk + 1) * ctas + chunks - 1, chunks)) - 1; }
};
__device__ __forceinline__ Shares make_shares(const AttnParams& p, int64_t chunks) {
    const int64_t most = p.share_min == 1 ? chunks : chunks / p.share_min;
    return {chunks, static_cast<int>(max(static_cast<int64_t>(1), min(most, static_cast<int64_t>(p.share_ctas))))};
}

// Tokens that a CTA of the step kernels with a 16-bit output may go through in one sum, or
// puts its sum by after: the tensor cores truncate as they add, so a sum over n tokens
// comes out about 6e-9 n too small, which an output's rounding (2^-11, fp16; 2^-8,
// bf16) has to cover. Of these tokens a warp adds up a quarter. (With every sum put
// by after 16384 tokens 32 sequences of 32768, 4-bit cache, 32/8 heads of 128 channels, bf16,
// took 242 us where they take 232, although none of their sums is that long.)
constexpr int kStepLong = 65536, kStepLongBf16 = 8 * kStepLong;

// Whether a CTA may go through more, of `chunks` at most that `ctas` share.
inline bool step_sums_long(int64_t chunks, int ctas, int share_min, int max_tokens, int out_dtype) {
    // Fewer CTAs share shorter lengths, of at least share_min chunks each.
    int64_t share = (chunks + ctas - 1) / ctas;
    if (share_min > 1 && share < 2 * static_cast<int64_t>(share_min)) share = 2 * static_cast<int64_t>(share_min);
    const int64_t tokens = share * kShareTokens;
    return (tokens < max_tokens ? tokens : max_tokens) > (out_dtype == AKV_Q_F16 ? kStepLong : kStepLongBf16);
}

struct ShareScratch {
    int64_t sums[32];
    int64_t before;
    int b;
};

// Counts all chunks with the whole CTA (ctas 0 when there are none).
__device__ __forceinline__ Shares count_shares(const AttnParams& p, int units, ShareScratch& sh) {
    int64_t n = 0;
    for (int b = threadIdx.x; b < p.c.B; b += blockDim.x) n += share_chunks(p, b);
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    if ((threadIdx.x & 31) == 0) sh.sums[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) n += sh.sums[w];
    Shares s = make_shares(p, n * units);
    if (n == 0) s.ctas = 0;
    return s;
}

// The sequence that chunk `at` belongs to, and the chunks before it.
__device__ __forceinline__ int find_sequence(const AttnParams& p, int64_t at, int units, ShareScratch& sh, int64_t& before) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        int64_t done = 0;
        bool found = false;
        for (int b0 = 0; b0 < p.c.B && !found; b0 += 32) {
            const int64_t n = b0 + lane < p.c.B ? static_cast<int64_t>(share_chunks(p, b0 + lane)) * units : 0;
            int64_t x = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (lane >= o) x += y;
            }
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, at < done + x);
            if (hit) {
                found = true;
                if (lane == __ffs(hit) - 1) {
                    sh.b = b0 + lane;
                    sh.before = done + x - n;
                }
            }
            done += __shfl_sync(0xFFFFFFFFu, x, 31);
        }
    }
    __syncthreads();
    before = sh.before;
    return sh.b;
}

// The partials of a row: part_ml[row(k)], k < n; `done` when its one piece
// wrote the row itself.
struct Parts {
    int n;
    bool done;
    int64_t first, rest, step;
    __device__ __forceinline__ int64_t row(int k) const { return k == 0 ? first : rest + k * step; }
};

// Chunks before sequence b and all chunks, by one warp (shares only).
__device__ __forceinline__ void warp_chunks(const AttnParams& p, int b, int64_t& before, int64_t& all) {
    const int lane = threadIdx.x & 31;
    before = all = 0;
    for (int i = lane; i < p.c.B; i += 32) {
        const int n = share_chunks(p, i);
        all += n;
        before += i < b ? n : 0;
    }
    for (int o = 16; o; o >>= 1) {
        all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
        before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    }
}

// Of row r of kv head h; by a whole warp.
__device__ __forceinline__ Parts find_parts(const AttnParams& p, int b, int h, int r) {
    const int bh = b * p.c.H + h;
    if (p.share_ctas == 0) {
        const int64_t first = static_cast<int64_t>(bh) * p.nsplits * p.R + r;
        return {p.nsplits, false, first, first, p.R};
    }
    if (p.share_ctas < 0) return {0, true, 0, 0, 0};
    int64_t before, chunks;
    warp_chunks(p, b, before, chunks);
    const int n = share_chunks(p, b);
    if (n == 0) return {0, true, 0, 0, 0};
    const int groups = (p.R + p.row_group - 1) / p.row_group, units = p.c.H * groups;
    const Shares s = make_shares(p, chunks * units);
    const int64_t at = before * units + static_cast<int64_t>(h * groups + r / p.row_group) * n;
    const int i0 = s.owner(at), i1 = s.owner(at + n - 1), rr = r % p.row_group;
    const int64_t step = 2 * static_cast<int64_t>(p.row_group), rest = i0 * step + rr;
    return {i1 - i0 + 1, i0 == i1, rest + (s.start(i0) == at ? 0 : p.row_group), rest, step};
}

// A row's sum of 2^score over its partials, sum * 2^top. The two stay apart
// where outputs are divided by it: as one number, top + log2 sum, a score of
// 1000 leaves 14 bits for the sum.
struct RowSum {
    float top, sum;  // -inf, 0: nothing seen; a NaN is in `sum`
    __device__ __forceinline__ bool none() const { return top == -CUDART_INF_F && !isnan(sum); }
    __device__ __forceinline__ float inverse() const { return none() ? 0.f : 1.f / sum; }
    __device__ __forceinline__ float lse() const { return isnan(sum) ? sum : none() ? top : top + log2f(sum); }
};

// By one warp; all lanes get it.
__device__ __forceinline__ RowSum combined_sum(const AttnParams& p, const Parts& parts) {
    const int lane = threadIdx.x & 31;
    float m = -CUDART_INF_F, l = 0.f;
    for (int s = lane; s < parts.n; s += 32) {
        const float2 v = p.part_ml[parts.row(s)];
        if (v.x == -CUDART_INF_F) continue;
        const float top = fmaxf(m, v.x);
        l = (m == -CUDART_INF_F ? 0.f : l * exp2f(m - top)) + v.y * exp2f(v.x - top);
        m = top;
    }
    float all = m;
    for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
    l = m == -CUDART_INF_F && !isnan(l) ? 0.f : l * exp2f(m - all);
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    return {all, l};
}

// Eight query rows as fragments of the second operand of S^T = K Q^T, in fp16
// after a power of two (fp32 rows in two parts), and the factor that turns
// their products with codes of scale 1 into base-2 scores; by one warp.
__device__ __forceinline__ void pack_rows(const AttnParams& p, int b, int h, int group) {
    const int lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3, r = 8 * group + g;
    const int steps = p.c.D <= 64 ? 4 : p.c.D <= 128 ? 8 : 16, parts = p.q_dtype == AKV_Q_F32 ? 2 : 1;
    const int64_t at = r < p.R ? q_row(p, b, h, r) : 0;
    uint32_t top = 0;
    for (int d = 16 * cc; d < p.c.D && r < p.R; d += 64) {
        float x[16];
        load_q16(p, at + d, x);
#pragma unroll
        for (int k = 0; k < 16; ++k) top = max(top, abs_bits(x[k]));
    }
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    const int e = row_exponent(__uint_as_float(top));
    const float up = power_of_two(e);
    const int64_t unit = static_cast<int64_t>(b * p.c.H + h) * ((p.R + 7) / 8) + group;
    uint2* to = p.q_rows + unit * steps * parts * 32 + lane;
    for (int j = 0; j < steps / 4; ++j) {
        const int d = 16 * cc + 64 * j;
        float x[16];
        if (d < p.c.D && r < p.R) {
            load_q16(p, at + d, x);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = x[4 * s + k] * up;
            const uint32_t h0 = pack_half2(y[0], y[1]), h1 = pack_half2(y[2], y[3]);
            to[(4 * j + s) * parts * 32] = make_uint2(h0, h1);
            if (parts == 2) to[((4 * j + s) * 2 + 1) * 32] = make_uint2(pack_rest(y[0], y[1], h0), pack_rest(y[2], y[3], h1));
        }
    }
    if (cc == 0) p.q_factors[unit * 8 + g] = p.c2 * power_of_two(-e);
}

// A row by one warp.
__device__ __forceinline__ void combine_row(const AttnParams& p, const Parts& parts, const RowSum& all, int64_t row) {
    const int lanes = p.c.D / 4;
    const float inv = all.inverse();
    for (int x = threadIdx.x & 31; x < lanes; x += 32) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < parts.n; s0 += 4) {
            float4 v[4];
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = s0 + k < parts.n ? p.part_ml[parts.row(s0 + k)].x : -CUDART_INF_F;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // What has seen nothing has no partial either.
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (f[k] != -CUDART_INF_F) v[k] = reinterpret_cast<const float4*>(p.part_o)[parts.row(s0 + k) * lanes + x];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float w = f[k] == -CUDART_INF_F ? 0.f : exp2f(f[k] - all.top);
                a.x = fmaf(v[k].x, w, a.x);
                a.y = fmaf(v[k].y, w, a.y);
                a.z = fmaf(v[k].z, w, a.z);
                a.w = fmaf(v[k].w, w, a.w);
            }
        }
        store4(p.out, p.out_dtype, row * p.c.D + 4 * x, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    }
}

// The first blocks: `rows` rows of the output, each its partials weighted
// by 2^(m - top), over the row's sum. Groups of D / 4 threads take every so many-th partial, four
// loads in flight each (the kernel is bound by load latency: with one thread
// per dimension 128 partials of 128 rows took 36 us); their sums are
// added in a fixed order. Where partials are few a warp does a row (by_warp).
// The other blocks: `packs` groups of eight query rows for the weights kernel,
// a warp each; or wtokens tokens of one kv head each: the stored scores of its rows become softmax weights, added up.
static __global__ void __launch_bounds__(kCombineThreads) combine_kernel(AttnParams p, int rows, bool by_warp, int wblocks, int wtokens, int packs) {
    __shared__ float lse[16];
    __shared__ int ends[16];
    __shared__ float w[kCombineThreads];
    __shared__ float4 part[kCombineThreads];
    const int tid = threadIdx.x;
    wait_for_previous_kernel();
    const int row_blocks = by_warp ? (rows + kCombineThreads / 32 - 1) / (kCombineThreads / 32) : rows;
    if (static_cast<int>(blockIdx.x) < row_blocks) {
        const int i = by_warp ? blockIdx.x * (kCombineThreads / 32) + (tid >> 5) : blockIdx.x;
        if (i >= rows) return;
        const int r = i % p.R, bh = i / p.R, h = bh % p.c.H, b = bh / p.c.H, D = p.c.D;
        const Parts parts = find_parts(p, b, h, r);  // every warp for itself
        if (parts.done) return;
        const RowSum all = combined_sum(p, parts);
        const int64_t row = out_row(p, b, h, r);
        if (by_warp ? (tid & 31) == 0 : tid == 0) {
            const float lse = all.lse();
            if (p.lse) p.lse[row] = lse;
            if (p.lse_out) p.lse_out[row] = lse * 0.69314718055994531f;
        }
        if (by_warp) {
            combine_row(p, parts, all, row);
            return;
        }
        const int lanes = D / 4, groups = kCombineThreads / lanes, x = tid % lanes, grp = tid / lanes;
        const float4* o = reinterpret_cast<const float4*>(p.part_o) + x;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < parts.n; s0 += kCombineThreads) {
            __syncthreads();
            if (s0 + tid < parts.n) {
                const float m = p.part_ml[parts.row(s0 + tid)].x;
                w[tid] = m == -CUDART_INF_F ? 0.f : exp2f(m - all.top);
            }
            __syncthreads();
            const int n = min(kCombineThreads, parts.n - s0);
            for (int s = grp; s < n && grp < groups; s += 4 * groups) {
                float4 v[4];
                float f[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int sk = s + k * groups;
                    f[k] = sk < n ? w[sk] : 0.f;
                    // A split that has nothing has no partial either.
                    v[k] = f[k] != 0.f ? o[parts.row(s0 + sk) * lanes] : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    a.x = fmaf(v[k].x, f[k], a.x);
                    a.y = fmaf(v[k].y, f[k], a.y);
                    a.z = fmaf(v[k].z, f[k], a.z);
                    a.w = fmaf(v[k].w, f[k], a.w);
                }
            }
        }
        part[tid] = a;
        __syncthreads();
        if (grp != 0) return;
        for (int k = 1; k < groups; ++k) {
            const float4 v = part[k * lanes + x];
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
        }
        const float inv = all.inverse();
        store4(p.out, p.out_dtype, row * D + 4 * x, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        return;
    }
    if (packs > 0) {
        const int i = (blockIdx.x - row_blocks) * (kCombineThreads / 32) + (tid >> 5), groups = (p.R + 7) / 8;
        if (i < packs) pack_rows(p, i / groups / p.c.H, i / groups % p.c.H, i % groups);
        return;
    }
    const int wb = blockIdx.x - row_blocks, bh = wb / wblocks, b = bh / p.c.H, t0 = wb % wblocks * wtokens;
    const int len = len_of(p, b), qlen = q_len_of(p, b);
    if (p.accumulate && t0 >= len) return;
    const int h = bh % p.c.H;
    for (int r = tid >> 5; r < p.R; r += kCombineThreads / 32) {
        const Parts parts = find_parts(p, b, h, r);
        const float v = parts.done ? p.lse[out_row(p, b, h, r)] : combined_sum(p, parts).lse();
        if ((tid & 31) == 0) {
            lse[r] = v;
            ends[r] = seen_by(p, r / p.G, len, qlen);
        }
    }
    __syncthreads();
    const float* sc = p.scores + static_cast<int64_t>(bh) * p.c.T * p.R;
    float* at = p.weights + static_cast<int64_t>(bh) * p.wstride;
    const int t_end = min(t0 + wtokens, p.c.T);
    for (int t = t0 + tid; t < t_end; t += 4 * kCombineThreads) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f}, old[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int tk = t + k * kCombineThreads;
            old[k] = p.accumulate && tk < min(t_end, len) ? at[tk] : 0.f;
        }
        if (p.R % 4 == 0) {
            for (int r = 0; r < p.R; r += 4) {
                float4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int tk = t + k * kCombineThreads;
                    v[k] = tk < min(t_end, len) ? *reinterpret_cast<const float4*>(sc + static_cast<int64_t>(tk) * p.R + r)
                                                : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int tk = t + k * kCombineThreads;
                    if (tk < ends[r]) sum[k] += exp2_fast(v[k].x - lse[r]);
                    if (tk < ends[r + 1]) sum[k] += exp2_fast(v[k].y - lse[r + 1]);
                    if (tk < ends[r + 2]) sum[k] += exp2_fast(v[k].z - lse[r + 2]);
                    if (tk < ends[r + 3]) sum[k] += exp2_fast(v[k].w - lse[r + 3]);
                }
            }
        } else {
            for (int r = 0; r < p.R; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int tk = t + k * kCombineThreads;
                    if (tk < min(ends[r], t_end)) sum[k] += exp2_fast(sc[static_cast<int64_t>(tk) * p.R + r] - lse[r]);
                }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int tk = t + k * kCombineThreads;
            if (tk < t_end && (!p.accumulate || tk < len)) at[tk] = old[k] + sum[k];
        }
    }
}

}  // namespace q8
}  // namespace akv
