// Store and restore of the 8-bit KV cache.
//
// Both move every element once. A thread holds pieces of 16 consecutive
// elements of a row: 16 bytes of codes, the widest access. Measured, 4 x 8192
// tokens, 8 heads, D 128, bf16 to int8: store 50 us, restore 38 us, each for
// 201 MB (4.0 and 5.3 TB/s; a copy's 6.42 would take 31 us). The store waits
// for its loads, then for the CTA's maximum; one element at a time the pair
// took 266 us.
#pragma once
#include "akv_q8_common.cuh"

namespace akv {
namespace q8 {

struct StoreParams {
    CacheDev c;
    const void* x[2];             // K, V rows
    int64_t xB[2], xT[2], xH[2];  // elements
    bool vec[2];                  // rows start on 16-byte boundaries
    const int32_t* start;
    const int32_t* counts;
    int n;
};

// Largest value of a CTA; `red` holds one word per warp.
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* red) {
    v = __reduce_max_sync(0xFFFFFFFFu, v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) v = max(v, red[w]);
    return v;
}

// 16 elements as they are in memory, and element i of them as a float.
template <typename T>
struct Piece {
    uint4 w[sizeof(T)];

    __device__ __forceinline__ void load(const T* at, bool vec) {
        if (vec) {
#pragma unroll
            for (int k = 0; k < static_cast<int>(sizeof(T)); ++k) w[k] = __ldg(reinterpret_cast<const uint4*>(at) + k);
        } else {
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (int k = 0; k < 16; ++k) e[k] = at[k];
        }
    }
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& v = w[i >> 2];
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
    // Bits of the largest |element|, as a float; an infinity or a NaN shows.
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t top = 0;
        if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, word(i) & 0x7FFFFFFFu);
        } else if (std::is_same<T, __nv_bfloat16>::value) {
            // The order of the magnitudes is that of their bits.
            uint32_t even = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                top = max(top, word(i) & 0x7FFF0000u);
                even = max(even, word(i) & 0x7FFFu);
            }
            top = max(top, even << 16);
        } else {
            __half2 m = __float2half2_rn(0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t v = word(i) & 0x7FFF7FFFu;
                m = __hmax2_nan(m, *reinterpret_cast<const __half2*>(&v));
            }
            const float2 f = __half22float2(m);
            top = max(abs_bits(f.x), abs_bits(f.y));
        }
        return top;
    }
    __device__ __forceinline__ float get(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(word(i));
        const uint32_t v = word(i >> 1);
        if (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? v & 0xFFFF0000u : v << 16);
        return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? v >> 16 : v)));
    }
};

// One CTA per (touched block, kv head, sequence x side). The new rows stay in
// registers (PP pieces a thread) between finding their largest value and
// coding them. Rows that a growing block holds already are read, coded again
// and written in place.
template <int FMT, typename T, int PP>
__global__ void __launch_bounds__(256, PP == 2 ? (sizeof(T) == 2 ? 6 : 4) : 1) store_kernel(StoreParams p) {
    __shared__ uint32_t red[8];
    const CacheDev& c = p.c;
    const int h = blockIdx.y, b = blockIdx.z >> 1, side = blockIdx.z & 1;
    const int start = p.start[b], count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    if (start < 0 || static_cast<int64_t>(start) + count > c.T) {
        // (No rows are nowhere outside. Asked here, so that both loads are in flight at a time.)
        if (count > 0 && threadIdx.x == 0 && blockIdx.x == 0) report(c.status, AKV_ERR_INVALID_ARGUMENT);
        if (start < 0 || start >= c.T) return;
    }
    const int end = start + min(count, c.T - start), shift = 31 - __clz(c.blk);
    const int64_t first_token = (static_cast<int64_t>(start >> shift) + blockIdx.x) << shift;  // of this block
    if (first_token >= end) return;
    const int block0 = static_cast<int>(first_token);
    const int first = max(start - block0, 0), last = min(end - block0, c.blk);  // rows [first, last) are new
    if (last <= first) return;
    int row0;
    const int phys = page_of(c, b, block0, row0);
    if (phys < 0) return;
    const SideDev& s = side ? c.v : c.k;
    uint8_t* codes = s.codes + code_offset(s, b, h, phys, row0);
    float* scale_at = s.scales + scale_offset(s, b, h, phys, row0 >> shift);
    const T* x = static_cast<const T*>(p.x[side]) + b * p.xB[side] + h * p.xH[side] + (block0 - start) * p.xT[side];
    const int64_t xT = p.xT[side];
    const int per_row = c.D / 16, pieces = (last - first) * per_row;
    Piece<T> v[PP];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < PP; ++k) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i >= pieces) break;
        const int r = first + i / per_row, d = i % per_row * 16;
        v[k].load(x + r * xT + d, p.vec[side]);
        top = max(top, v[k].largest());
    }
    float had = first > 0 ? *scale_at : 0.f;
    top = cta_max(top, red);  // its barrier: everyone has read the scale
    float scale = block_scale<FMT>(top);
    if (first > 0) {
        if (scale <= had || isnan(had)) {
            scale = had;
        } else {
            // The rows that are there already, under the larger scale.
            const float inv = block_inverse(scale);
            for (int i = threadIdx.x; i < first * per_row; i += blockDim.x) {
                uint4* at = reinterpret_cast<uint4*>(codes + (i / per_row) * s.sT + i % per_row * 16);
                uint4 w = *at;
                uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float f[4];
                    from_codes4<FMT>(u[k], f);
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[j] = __fmul_rn(__fmul_rn(f[j], had), inv);
                    u[k] = to_codes4<FMT>(f);
                }
                *at = w;
            }
        }
    }
    const float inv = block_inverse(scale);
    // A block with a NaN scale holds zeros: a NaN code would meet the softmax
    // weight 0 of rows that do not see it, in the attention's products.
    if (isnan(scale)) {
#pragma unroll
        for (int k = 0; k < PP; ++k)
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(T)); ++j) v[k].w[j] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < PP; ++k) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i >= pieces) break;
        const int r = first + i / per_row, d = i % per_row * 16;
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(v[k].get(4 * j + e), inv);
            u[j] = to_codes4<FMT>(f);
        }
        *reinterpret_cast<uint4*>(codes + r * s.sT + d) = make_uint4(u[0], u[1], u[2], u[3]);
    }
    if (threadIdx.x == 0) *scale_at = scale;
}

struct RestoreParams {
    CacheDev c;
    void* out[2];
    const int32_t* start;
    int n;
};

// One thread per piece, in the order of the output; grid.y: sequence x side.
template <int FMT, typename T>
__global__ void __launch_bounds__(256) restore_kernel(RestoreParams p) {
    const CacheDev& c = p.c;
    const int b = blockIdx.y >> 1, side = blockIdx.y & 1;
    const SideDev& s = side ? c.v : c.k;
    const unsigned per_row = c.D / 16, per_token = per_row * c.H;
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= per_token * p.n) return;
    const unsigned ti = i / per_token, rest = i - ti * per_token;
    const int h = rest / per_row, d = (rest - h * per_row) * 16;
    wait_for_previous_kernel();
    const int64_t t = static_cast<int64_t>(ti) + (p.start ? p.start[b] : 0);
    int row = 0;
    const int phys = t >= 0 && t < c.T ? page_of(c, b, static_cast<int>(t), row) : -1;
    uint4 w = make_uint4(0, 0, 0, 0);
    float scale = 0.f;
    if (phys >= 0) {
        w = *reinterpret_cast<const uint4*>(s.codes + code_offset(s, b, h, phys, row) + d);
        scale = s.scales[scale_offset(s, b, h, phys, row >> (31 - __clz(c.blk)))];
    }
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t o[4 * sizeof(T)];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float f[4];
        from_codes4<FMT>(u[k], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __fmul_rn(f[j], scale);
        if (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[sizeof(T) == 4 ? 4 * k + j : 0] = __float_as_uint(f[j]);
        } else {
            o[2 * k] = pack2<T>(f[0], f[1]);
            o[2 * k + 1] = pack2<T>(f[2], f[3]);
        }
    }
    uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out[side]) + (static_cast<int64_t>(b) * p.n * per_token + i) * 16);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T)); ++k) out[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
}

}  // namespace q8
}  // namespace akv
