// Store and restore of the 8-bit KV cache.
#pragma once
#include "akv_q8_common.cuh"

namespace akv {
namespace q8 {

constexpr int kStoreThreads = 256;

struct StoreParams {
    CacheDev c;
    const void* x[2];       // K, V rows
    int64_t xB[2], xT[2], xH[2];  // elements
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

// One CTA per (touched block, kv head, sequence x side). Reads its rows twice
// (the second time from L1/L2): once for the largest value, once to code.
template <int FMT, typename T>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(StoreParams p) {
    __shared__ uint32_t red[kStoreThreads / 32];
    const CacheDev& c = p.c;
    const int h = blockIdx.y, b = blockIdx.z >> 1, side = blockIdx.z & 1;
    const int64_t start = p.start[b];
    const int64_t count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    if (start < 0 || start + count > c.T) {
        if (threadIdx.x == 0 && blockIdx.x == 0) report(c.status, AKV_ERR_INVALID_ARGUMENT);
        if (start < 0) return;
    }
    const int64_t end = min(start + count, static_cast<int64_t>(c.T));
    const int64_t block0 = (start / c.blk + blockIdx.x) * c.blk;  // first token of this block
    const int first = static_cast<int>(max(start, block0) - block0);  // rows [first, last) are new
    const int last = static_cast<int>(min(end - block0, static_cast<int64_t>(c.blk)));
    if (last <= first) return;
    const int phys = page_of(c, b, static_cast<int>(block0));
    if (phys < 0) return;
    const SideDev& s = side ? c.v : c.k;
    const int row0 = static_cast<int>(block0 % c.P);
    uint8_t* codes = s.codes + code_offset(s, b, h, phys, row0);
    float* scale_at = s.scales + scale_offset(s, b, h, phys, row0 / c.blk);
    const T* x = static_cast<const T*>(p.x[side]) + b * p.xB[side] + h * p.xH[side] + (block0 - start) * p.xT[side];
    const int64_t xT = p.xT[side];
    const int n = (last - first) * c.D;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < n; i += kStoreThreads) top = max(top, abs_bits(to_f32(x[(first + i / c.D) * xT + i % c.D])));
    top = cta_max(top, red);
    float scale = block_scale<FMT>(top);
    if (first > 0) {
        const float had = *scale_at;
        __syncthreads();  // everyone has read it
        if (!(scale <= had)) {
            if (!isnan(had)) {
                // The rows that are there already, under the larger scale.
                const float inv = block_inverse(scale);
                for (int i = threadIdx.x; i < first * c.D; i += kStoreThreads) {
                    uint8_t* at = codes + (i / c.D) * s.sT + i % c.D;
                    *at = to_code<FMT>(__fmul_rn(__fmul_rn(from_code<FMT>(*at), had), inv));
                }
            } else {
                scale = had;
            }
        } else {
            scale = had;
        }
    }
    const float inv = block_inverse(scale);
    for (int i = threadIdx.x; i < n; i += kStoreThreads) {
        const int r = first + i / c.D, d = i % c.D;
        codes[r * s.sT + d] = to_code<FMT>(__fmul_rn(to_f32(x[r * xT + d]), inv));
    }
    if (threadIdx.x == 0) *scale_at = scale;
}

struct RestoreParams {
    CacheDev c;
    void* out[2];
    const int32_t* start;
    int n;
};

// One thread per 16 codes, in the order of the output.
template <int FMT, typename T>
__global__ void __launch_bounds__(256) restore_kernel(RestoreParams p) {
    const CacheDev& c = p.c;
    const int side = blockIdx.y;
    const SideDev& s = side ? c.v : c.k;
    const int per_row = c.D / 16;
    const int64_t total = static_cast<int64_t>(c.B) * p.n * c.H * per_row;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int d16 = static_cast<int>(i % per_row);
    const int64_t rowi = i / per_row;
    const int h = static_cast<int>(rowi % c.H);
    const int64_t bt = rowi / c.H;
    const int b = static_cast<int>(bt / p.n);
    const int64_t t = bt % p.n + (p.start ? p.start[b] : 0);
    __align__(16) T o[16];
    const int phys = t >= 0 && t < c.T ? page_of(c, b, static_cast<int>(t)) : -1;
    if (phys < 0) {
        for (int k = 0; k < 16; ++k) o[k] = from_f32<T>(0.f);
    } else {
        const int row = static_cast<int>(t % c.P);
        const uint4 w = *reinterpret_cast<const uint4*>(s.codes + code_offset(s, b, h, phys, row) + d16 * 16);
        const float scale = s.scales[scale_offset(s, b, h, phys, row / c.blk)];
        const uint8_t* q = reinterpret_cast<const uint8_t*>(&w);
        for (int k = 0; k < 16; ++k) o[k] = from_f32<T>(__fmul_rn(from_code<FMT>(q[k]), scale));
    }
    uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out[side]) + i * 16);
    for (int k = 0; k < static_cast<int>(sizeof(T)); ++k) out[k] = reinterpret_cast<const uint4*>(o)[k];
}

}  // namespace q8
}  // namespace akv
