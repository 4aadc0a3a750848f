// Eviction from the 8-bit KV cache by accumulated attention weight.
#pragma once
#include "akv_q8_common.cuh"
#include "akv_q8_store.cuh"

namespace akv {
namespace q8 {

constexpr int kSelectThreads = 1024;

struct EvictParams {
    CacheDev src, dst;
    const float* weights;
    int64_t wstride;
    const int32_t* lens;
    int keep, sinks, recent;
    int32_t* kept;
    int32_t* out_lens;
    float* out_weights;
    int64_t ostride;
};

// Weights in an order of unsigned numbers: negative below positive, -0 equal
// to 0, a NaN above everything.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (isnan(w)) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the CTA's threads before this one; `total` gets the sum of all.
__device__ __forceinline__ int cta_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sums[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xFFFFFFFFu, s, o);
            if (lane >= o) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    *total = warp_sums[31];
    return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// One CTA per (kv head, sequence). The middle tokens' cut-off is found one
// byte of the key at a time, by a histogram of the keys that still agree with
// the bytes found; then one pass in order writes what lies above it, and of
// what equals it the first few.
__global__ void __launch_bounds__(kSelectThreads) select_kernel(EvictParams p) {
    __shared__ int hist[256];
    __shared__ int sums[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int64_t unit = static_cast<int64_t>(b) * p.src.H + h;
    const float* w = p.weights + unit * p.wstride;
    int32_t* kept = p.kept + unit * p.keep;
    float* ow = p.out_weights + unit * p.ostride;
    const int len = p.lens ? min(max(p.lens[b], 0), p.src.T) : p.src.T;
    const int n = min(len, p.keep);
    if (h == 0 && tid == 0) p.out_lens[b] = n;
    for (int i = n + tid; i < p.keep; i += kSelectThreads) {
        kept[i] = -1;
        ow[i] = 0.f;
    }
    if (len <= p.keep) {
        for (int i = tid; i < n; i += kSelectThreads) {
            kept[i] = i;
            ow[i] = w[i];
        }
        return;
    }
    const int lo = p.sinks, hi = len - p.recent;
    uint32_t prefix = 0;
    int want = p.keep - p.sinks - p.recent;  // of the tokens whose key agrees with `prefix` so far
    for (int shift = 24; want > 0 && shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int t = lo + tid; t < hi; t += kSelectThreads) {
            const uint32_t k = order_key(w[t]);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255, left = want;
            while (left > hist[d]) left -= hist[d--];
            s_prefix = prefix | static_cast<uint32_t>(d) << shift;
            s_want = left;
        }
        __syncthreads();
        prefix = s_prefix;
        want = s_want;
    }
    const bool none = p.keep == p.sinks + p.recent;
    int out = 0, equal = 0;
    for (int t0 = 0; t0 < len; t0 += kSelectThreads) {
        const int t = t0 + tid;
        const bool in = t < len, fixed = in && (t < lo || t >= hi);
        const float x = in ? w[t] : 0.f;
        const uint32_t k = order_key(x);
        const bool same = in && !fixed && !none && k == prefix;
        int total, all;
        const int before = equal + cta_scan(same, sums, &all);
        const bool take = fixed || (in && !none && (k > prefix || (same && before < want)));
        const int at = out + cta_scan(take, sums, &total);
        if (take) {
            kept[at] = t;
            ow[at] = x;
        }
        equal += all;
        out += total;
    }
}

// One CTA per (block of the new cache, kv head, sequence x side).
template <int FMT>
__global__ void __launch_bounds__(256) pack_kernel(EvictParams p) {
    __shared__ uint32_t red[8];
    const CacheDev &a = p.src, &c = p.dst;
    const int h = blockIdx.y, b = blockIdx.z >> 1, side = blockIdx.z & 1;
    const SideDev &from = side ? a.v : a.k, &to = side ? c.v : c.k;
    const int64_t unit = static_cast<int64_t>(b) * a.H + h;
    const int32_t* kept = p.kept + unit * p.keep;
    const int row0 = blockIdx.x * c.blk;
    const int n = min(p.out_lens[b] - row0, c.blk);
    if (n <= 0) return;
    const int phys = page_of(c, b, row0);
    if (phys < 0) return;
    auto value = [&](int r, int d) {
        const int t = kept[row0 + r], pg = page_of(a, b, t), row = t % a.P;
        if (pg < 0) return 0.f;
        return __fmul_rn(from_code<FMT>(from.codes[code_offset(from, b, h, pg, row) + d]),
                         from.scales[scale_offset(from, b, h, pg, row / a.blk)]);
    };
    uint32_t top = 0;
    for (int i = threadIdx.x; i < n * c.D; i += 256) top = max(top, abs_bits(value(i / c.D, i % c.D)));
    const float scale = block_scale<FMT>(cta_max(top, red)), inv = block_inverse(scale);
    const int in_page = row0 % c.P;
    uint8_t* codes = to.codes + code_offset(to, b, h, phys, in_page);
    for (int i = threadIdx.x; i < c.blk * c.D; i += 256) {
        const int r = i / c.D, d = i % c.D;
        codes[r * to.sT + d] = r < n ? to_code<FMT>(__fmul_rn(value(r, d), inv)) : 0;
    }
    if (threadIdx.x == 0) to.scales[scale_offset(to, b, h, phys, in_page / c.blk)] = scale;
}

}  // namespace q8
}  // namespace akv
