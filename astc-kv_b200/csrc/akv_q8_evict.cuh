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
    int columns;                // weights per row to be written, at least keep
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

// One CTA per (kv head, sequence). The middle tokens' cut-off is the key of
// the last one that stays; it is found 11, 11 and 10 bits at a time, by a
// histogram of the keys that agree with the bits found. Then votes give every
// kept token its place among its warp's (keys above the cut-off, and of the
// equal ones the first few of the row), and a scan over the warps the rest.
//
// A warp has a run of the row of its own and a lane every 32nd token of it, of
// which it keeps HELD weights in registers; of rows of more than 1024 x HELD
// the rest is read again in every pass, from L2. (HELD 8 for caches of up to
// 8192 tokens: an eviction of 8192 to 1001 tokens takes 17 us with its restore, 25 us with
// the code unrolled for 32.) Measured, 256 rows of 841
// to 32768 weights: 40 us; reading the row in each of five passes 70 us.
template <int HELD>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(EvictParams p) {
    __shared__ int hist[2048];
    __shared__ int sums[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t unit = static_cast<int64_t>(b) * p.src.H + h;
    const float* w = p.weights + unit * p.wstride;
    int32_t* kept = p.kept + unit * p.keep;
    float* ow = p.out_weights + unit * p.ostride;
    const int len = p.lens ? min(max(p.lens[b], 0), p.src.T) : p.src.T;
    const int n = min(len, p.keep);
    allow_next_kernel();
    if (h == 0 && tid == 0) p.out_lens[b] = n;
    for (int i = n + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
    for (int i = n + tid; i < p.columns; i += kSelectThreads) ow[i] = 0.f;
    if (len <= p.keep) {
        for (int i = tid; i < n; i += kSelectThreads) {
            kept[i] = i;
            ow[i] = w[i];
        }
        return;
    }
    const int lo = p.sinks, hi = len - p.recent;
    const int rounds = (len + kSelectThreads - 1) / kSelectThreads;  // of a warp's run, 32 tokens each
    const int t0 = warp * rounds * 32 + lane;
    float held[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) held[k] = k < rounds && t0 + 32 * k < len ? w[t0 + 32 * k] : 0.f;
    // Calls f with the token and its weight, in order, every lane of the warp
    // alike; tokens from len on are not there.
    auto for_tokens = [&](auto f) {
#pragma unroll
        for (int k = 0; k < HELD; ++k)
            if (k < rounds) f(t0 + 32 * k, held[k]);
        for (int k = HELD; k < rounds; ++k) f(t0 + 32 * k, t0 + 32 * k < len ? w[t0 + 32 * k] : 0.f);
    };
    uint32_t prefix = 0;
    int want = p.keep - p.sinks - p.recent;  // of the tokens whose key agrees with `prefix` so far
    const bool none = want == 0;
    for (int pass = 0; pass < 3 && !none; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t mask = pass == 2 ? 1023u : 2047u;
        hist[tid] = hist[tid + kSelectThreads] = 0;
        __syncthreads();
        int zeros = 0;  // tokens that never received weight are many: one bin
        for_tokens([&](int t, float x) {
            const uint32_t key = order_key(x);
            if (t < lo || t >= hi) return;
            if (pass == 0 && key == 0x80000000u) ++zeros;
            else if (pass == 0 || ((key ^ prefix) >> (shift + (pass == 1 ? 11 : 10))) == 0) atomicAdd(&hist[(key >> shift) & mask], 1);
        });
        zeros = __reduce_add_sync(0xFFFFFFFFu, zeros);
        if (zeros && lane == 0) atomicAdd(&hist[0x80000000u >> 21], zeros);
        __syncthreads();
        // Bins from the highest down, two a thread.
        const int d = 2047 - 2 * tid, upper = hist[d], lower = hist[d - 1];
        int total;
        const int before = cta_scan(upper + lower, sums, &total);
        if (before < want && want <= before + upper + lower) {
            const bool first = want <= before + upper;
            s_prefix = prefix | static_cast<uint32_t>(first ? d : d - 1) << shift;
            s_want = want - before - (first ? 0 : upper);
        }
        __syncthreads();
        prefix = s_prefix;
        want = s_want;
    }
    // What a token is: kept for its place or its key, or equal to the cut-off.
    auto kind = [&](int t, float x, bool& above, bool& equal) {
        const uint32_t key = order_key(x);
        const bool in = t < len, fixed = in && (t < lo || t >= hi);
        above = fixed || (in && !none && key > prefix);
        equal = in && !fixed && !none && key == prefix;
    };
    int above = 0, equal = 0;  // of the warp's run
    for_tokens([&](int t, float x) {
        bool a, e;
        kind(t, x, a, e);
        above += __popc(__ballot_sync(0xFFFFFFFFu, a));
        equal += __popc(__ballot_sync(0xFFFFFFFFu, e));
    });
    int total;
    int left = want - cta_scan(lane == 0 ? equal : 0, sums, &total);  // equal ones that the run may keep
    left = __shfl_sync(0xFFFFFFFFu, left, 0);
    const int take = max(0, min(equal, left));
    int at = cta_scan(lane == 0 ? above + take : 0, sums, &total);
    at = __shfl_sync(0xFFFFFFFFu, at, 0);
    const uint32_t below = (1u << lane) - 1;
    for_tokens([&](int t, float x) {
        bool a, e;
        kind(t, x, a, e);
        const uint32_t equals = __ballot_sync(0xFFFFFFFFu, e);
        const bool in = a || (e && __popc(equals & below) < left);
        const uint32_t ins = __ballot_sync(0xFFFFFFFFu, in);
        if (in) {
            const int place = at + __popc(ins & below);
            kept[place] = t;
            ow[place] = x;
        }
        at += __popc(ins);
        left -= __popc(equals);
    });
}

// Largest |code| of four, as fp16 (exact; a NaN code stays one).
template <int FMT>
__device__ __forceinline__ __half2 max_of_codes(uint32_t w, __half2 m) {
    uint32_t lo, hi;
    codes_to_half<FMT>(w, lo, hi);
    m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&lo)));
    return __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&hi)));
}

// One CTA per (block of the new cache, kv head, sequence), K and V together:
// the kept tokens and their pages are looked up once, and both sides' rows are
// in flight at a time. The rows' codes stay in registers (PP pieces of 16 a
// thread and side) between finding the largest value and coding them under
// the new scale. Measured, 32 ragged sequences to 4096 tokens, 8 heads, D 128,
// e4m3: 105 us for 367 MB (3.5 TB/s); K and V in CTAs of their own 167 us.
template <int FMT, int PP>
__global__ void __launch_bounds__(256, PP == 2 ? 6 : 2) pack_kernel(EvictParams p) {
    __shared__ uint32_t red[2][8];
    const CacheDev &a = p.src, &c = p.dst;
    const int h = blockIdx.y, b = blockIdx.z;
    const int32_t* kept = p.kept + (static_cast<int64_t>(b) * a.H + h) * p.keep;
    const int row0 = blockIdx.x * c.blk, per_row = c.D / 16;
    const int len = p.lens ? min(max(p.lens[b], 0), a.T) : a.T;
    const int n = min(min(len, p.keep) - row0, c.blk);
    int in_page;
    const int phys = n > 0 ? page_of(c, b, row0, in_page) : -1;
    // For the kept tokens; and in a CTA of each row at least, so that the
    // kernel does not end before the selection (the next one waits for this
    // one alone).
    if (phys >= 0 || blockIdx.x == 0) wait_for_previous_kernel();
    if (phys < 0) return;
    uint4 w[2][PP];
    float sc[2][PP];
#pragma unroll
    for (int k = 0; k < PP; ++k) {
        const int i = threadIdx.x + k * 256, r = i / per_row;
        w[0][k] = w[1][k] = make_uint4(0, 0, 0, 0);
        sc[0][k] = sc[1][k] = 0.f;
        if (r >= n) continue;
        int row;
        const int pg = page_of(a, b, kept[row0 + r], row);
        if (pg < 0) continue;
        const int piece = i - r * per_row;
        w[0][k] = __ldg(reinterpret_cast<const uint4*>(a.k.codes + code_offset(a.k, b, h, pg, row)) + piece);
        w[1][k] = __ldg(reinterpret_cast<const uint4*>(a.v.codes + code_offset(a.v, b, h, pg, row)) + piece);
        sc[0][k] = a.k.scales[scale_offset(a.k, b, h, pg, row / a.blk)];
        sc[1][k] = a.v.scales[scale_offset(a.v, b, h, pg, row / a.blk)];
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < PP; ++k) {
            __half2 m = __float2half2_rn(0.f);
            m = max_of_codes<FMT>(w[side][k].x, m);
            m = max_of_codes<FMT>(w[side][k].y, m);
            m = max_of_codes<FMT>(w[side][k].z, m);
            m = max_of_codes<FMT>(w[side][k].w, m);
            const float2 f = __half22float2(m);
            // Rounding keeps the order: the largest code gives the largest value.
            top = max(top, max(abs_bits(__fmul_rn(f.x, sc[side][k])), abs_bits(__fmul_rn(f.y, sc[side][k]))));
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        if ((threadIdx.x & 31) == 0) red[side][threadIdx.x >> 5] = top;
    }
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const SideDev& to = side ? c.v : c.k;
        uint32_t top = red[side][0];
#pragma unroll
        for (int k = 1; k < 8; ++k) top = max(top, red[side][k]);
        const float scale = block_scale<FMT>(top), inv = block_inverse(scale);
        if (isnan(scale)) {  // see store_kernel
#pragma unroll
            for (int k = 0; k < PP; ++k) {
                w[side][k] = make_uint4(0, 0, 0, 0);
                sc[side][k] = 0.f;
            }
        }
        uint8_t* codes = to.codes + code_offset(to, b, h, phys, in_page);
#pragma unroll
        for (int k = 0; k < PP; ++k) {
            const int i = threadIdx.x + k * 256, r = i / per_row;
            if (r >= c.blk) break;
            uint32_t u[4] = {w[side][k].x, w[side][k].y, w[side][k].z, w[side][k].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[4];
                from_codes4<FMT>(u[j], f);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(__fmul_rn(f[e], sc[side][k]), inv);
                u[j] = to_codes4<FMT>(f);
            }
            reinterpret_cast<uint4*>(codes + r * to.sT)[i - r * per_row] = make_uint4(u[0], u[1], u[2], u[3]);
        }
        if (threadIdx.x == 0) to.scales[scale_offset(to, b, h, phys, in_page / c.blk)] = scale;
    }
}

}  // namespace q8
}  // namespace akv
