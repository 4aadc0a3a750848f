// 4-bit KV cache: kernel-side view of an AkvQ4Cache, code conversions.
#pragma once
#include "../../include/akv_q4.h"
#include "akv_q8_common.cuh"

namespace akv {
namespace q4 {

struct SideDev {
    uint8_t* codes;
    __half* scales;
    int64_t sB, sH, sP, sT;      // bytes
    int64_t cB, cH, cP, cG;      // scales, elements
};

struct CacheDev {
    SideDev k, v;
    const int32_t* table;
    int B, H, D, T, P, pps, num_pages;
    int page_shift;              // log2 of P, 31 where one page holds every token, -1 otherwise
    int32_t* status;
};

inline SideDev to_dev(const AkvQ4Side& s) {
    return {static_cast<uint8_t*>(s.codes), static_cast<__half*>(s.scales), s.stride_batch, s.stride_head, s.stride_page, s.stride_token,
            s.scale_stride_batch, s.scale_stride_head, s.scale_stride_page, s.scale_stride_group};
}

inline CacheDev to_dev(const AkvQ4Cache& c) {
    CacheDev d;
    d.k = to_dev(c.k);
    d.v = to_dev(c.v);
    d.table = c.block_table_dev;
    d.B = c.batch; d.H = c.kv_heads; d.D = c.head_dim; d.T = c.max_tokens; d.P = c.page_tokens;
    d.pps = c.pages_per_seq; d.num_pages = c.num_pages;
    d.status = c.status_dev;
    d.page_shift = c.page_tokens >= c.max_tokens ? 31 : -1;
    for (int i = 4; i < 31 && d.page_shift < 0; ++i)
        if (c.page_tokens == 1 << i) d.page_shift = i;
    return d;
}

// Physical page of token t (0 <= t < T) of sequence b and the token's row in
// it; -1 for a table entry outside the pool.
__device__ __forceinline__ int page_of(const CacheDev& c, int b, int t, int& row) {
    const int p = c.page_shift >= 0 ? t >> c.page_shift : t / c.P;
    row = t - p * c.P;
    if (!c.table) return p;
    const int v = __ldg(c.table + static_cast<int64_t>(b) * c.pps + p);
    if (static_cast<unsigned>(v) >= static_cast<unsigned>(c.num_pages)) {
        q8::report(c.status, AKV_ERR_BAD_BLOCK_TABLE);
        return -1;
    }
    return v;
}

__device__ __forceinline__ int64_t code_offset(const SideDev& s, int b, int h, int phys, int row) {
    return b * s.sB + h * s.sH + phys * s.sP + row * s.sT;
}
// Of group 0.
__device__ __forceinline__ int64_t scale_offset(const SideDev& s, int b, int h, int phys, int row) {
    return b * s.cB + h * s.cH + phys * s.cP + row;
}

// Eight codes as four fp16 pairs, exactly (a conversion takes 3.6 cycles a warp in a
// loop of its own; moving sign, exponent and mantissa bits into place would be four integer
// instructions a pair instead).
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\ncvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

// The nearest codes of eight numbers, ties to even, beyond 6 to 6.
__device__ __forceinline__ uint32_t to_codes(const float (&y)[8]) {
    uint32_t w;
    asm("{\n.reg .b8 a, b, c, d;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\nmov.b32 %0, {a, b, c, d};\n}\n"
        : "=r"(w) : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// The largest scale: 6 times it is the largest multiple of 6 powers of two
// that fp16 holds, 65472.
constexpr float kMostScale = 10912.f;

// x / scale rounded to nearest, given the scale's approximate reciprocal (a
// unit in the last place off at most): the estimate q of the quotient and one
// correction by its remainder, which is exact (Markstein). q + remainder *
// inverse is then off by 2^-45 of itself before its one rounding, and a
// quotient of 24 bits by 11 is 2^-36 away at least from what would round
// another way. Ties between two codes have to be seen as ties: a 16-bit x is
// often a small multiple of the scale. 0 for a scale of 0.
__device__ __forceinline__ float quotient(float x, float scale, float inverse) {
    const float q = __fmul_rn(x, inverse);
    return __fmaf_rn(__fmaf_rn(-q, scale, x), inverse, q);
}
__device__ __forceinline__ float inverse_of(float scale) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(scale));
    return scale > 0.f ? y : 0.f;
}

}  // namespace q4
}  // namespace akv
