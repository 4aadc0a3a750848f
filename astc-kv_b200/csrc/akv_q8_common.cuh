// 8-bit KV cache: kernel-side view of an AkvQ8Cache, code conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>

#include "../../include/akv_q8.h"

namespace akv {
namespace q8 {

struct SideDev {
    uint8_t* codes;
    float* scales;
    int64_t sB, sH, sP, sT;  // bytes
    int64_t cB, cH, cP;      // scales, elements
};

struct CacheDev {
    SideDev k, v;
    const int32_t* table;
    int B, H, D, T, P, pps, num_pages, blk, fmt;
    int page_shift;          // log2 of P, 31 where one page holds every token, -1 otherwise
    int32_t* status;
};

inline SideDev to_dev(const AkvQ8Side& s) {
    return {static_cast<uint8_t*>(s.codes), s.scales, s.stride_batch, s.stride_head, s.stride_page, s.stride_token,
            s.scale_stride_batch, s.scale_stride_head, s.scale_stride_page};
}

inline CacheDev to_dev(const AkvQ8Cache& c) {
    CacheDev d;
    d.k = to_dev(c.k);
    d.v = to_dev(c.v);
    d.table = c.block_table_dev;
    d.B = c.batch; d.H = c.kv_heads; d.D = c.head_dim; d.T = c.max_tokens; d.P = c.page_tokens;
    d.pps = c.pages_per_seq; d.num_pages = c.num_pages; d.blk = c.block_tokens; d.fmt = c.format;
    d.status = c.status_dev;
    d.page_shift = c.page_tokens >= c.max_tokens ? 31 : -1;
    for (int i = 4; i < 31 && d.page_shift < 0; ++i)
        if (c.page_tokens == 1 << i) d.page_shift = i;
    return d;
}

// Ordering with the kernel before or after on the stream when both are
// launched as programmatic dependents (no effect otherwise): the next one may
// be brought onto the SMs, and wait until everything before has finished. A
// kernel waits in one CTA at least, whatever it has to do, since its end is
// all that the next one's wait sees.
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void report(int32_t* status, int code) {
    if (status) atomicExch(status, code);
}

// Physical page of token t (0 <= t < T) of sequence b and the token's row in
// it; -1 for a table entry outside the pool.
__device__ __forceinline__ int page_of(const CacheDev& c, int b, int t, int& row) {
    const int p = c.page_shift >= 0 ? t >> c.page_shift : t / c.P;
    row = t - p * c.P;
    if (!c.table) return p;
    const int v = __ldg(c.table + static_cast<int64_t>(b) * c.pps + p);
    if (static_cast<unsigned>(v) >= static_cast<unsigned>(c.num_pages)) {
        report(c.status, AKV_ERR_BAD_BLOCK_TABLE);
        return -1;
    }
    return v;
}

__device__ __forceinline__ int64_t code_offset(const SideDev& s, int b, int h, int phys, int row) {
    return b * s.sB + h * s.sH + phys * s.sP + row * s.sT;
}

__device__ __forceinline__ int64_t scale_offset(const SideDev& s, int b, int h, int phys, int block) {
    return b * s.cB + h * s.cH + phys * s.cP + block;
}

// Four codes as floats, exactly.
template <int FMT>
__device__ __forceinline__ void from_codes4(uint32_t w, float (&x)[4]) {
    if (FMT == AKV_Q8_INT8) {
        // code + 128 in the low byte of 2^23, less 2^23 + 128.
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 | k)) - 8388736.f;
    } else {
        const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFF), __NV_E4M3));
        const __half2 b = __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3));
        const float2 f = __half22float2(a), g = __half22float2(b);
        x[0] = f.x; x[1] = f.y; x[2] = g.x; x[3] = g.y;
    }
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

// Codes of four y = x / scale with |y| <= M up to rounding (M = 127 or 448).
template <int FMT>
__device__ __forceinline__ uint32_t to_codes4(const float (&y)[4]) {
    if (FMT == AKV_Q8_INT8) {
        // The sum with 1.5 * 2^23 rounds to the nearest whole number, ties to
        // even; its low byte is that number's.
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = __float_as_uint(__fadd_rn(y[k], 12582912.f));
        return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    }
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3)) << 16;
}

// Scale of a block from the largest |x| of its rows, given as the bits of
// |x| (so that an infinity or a NaN, whose bits exceed every number's, is
// seen): amax / M as a product with 1/M; NaN for what is not finite, 0 where
// the scale would be subnormal (its reciprocal could overflow).
template <int FMT>
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    constexpr float inv_most = FMT == AKV_Q8_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f;
    const float s = __fmul_rn(__uint_as_float(amax_bits), inv_most);
    return s < 1.17549435e-38f ? 0.f : s;
}

// 1 / scale; 0 for a block of zeros or one that holds no numbers.
__device__ __forceinline__ float block_inverse(float scale) { return scale > 0.f ? __frcp_rn(scale) : 0.f; }

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Two floats as a pair of a 16-bit type.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace q8
}  // namespace akv
