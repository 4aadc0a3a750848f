// Append and restore of the 4-bit KV cache.
//
// Both move each value once: 4 bytes of two 16-bit values in and 9 bits out, or the
// other way, so memory bounds them where tokens are many, and the launch where
// they are few.
//
// append_kernel: a lane holds eight consecutive channels of a token's head: 16
// bytes of 16-bit rows in, one word of codes out, and four lanes share a scale. The
// other half of its rotated pairs is loaded a second time by this lane, with the
// same loads, which ask L1 not to keep lines (rows meet no barrier and no shared memory). A lane keeps its
// token's cosines and sines for all heads that it goes through.
// append_pairs_kernel: both halves of eight pairs a lane, see there.
//
// Measured with 8 heads of 128 channels, bf16, rotated, 4 x 8192 tokens (134 MB
// in, 38 MB out): pairs 41 to 43 us, 4.2 TB/s, 64 % of a copy's rate, with no unit full
// (issue 47 % of the cycles, DRAM 24 %, 20 % of the warps that an SM can hold; 36 us
// without rotation); the general kernel 66 to 68 interleaved and 70 to 72 with 96 channels.
// With 32 query heads 128 to 132.
// One token of 64 sequences 3.4 us. Restore of the 4 x 8192 tokens 36 us, 4.8 TB/s (no unit
// full: issue 64 %, DRAM 36 %).
#pragma once
#include "akv_q4_common.cuh"
#include "akv_rotary.cuh"

namespace akv {
namespace q4 {

struct AppendParams {
    CacheDev c;
    RotaryDev r;
    const void* x[3];             // K, V, Q rows
    int64_t xB[3], xT[3], xH[3];  // elements
    void* q_out;
    const int32_t* start;
    const int32_t* counts;
    const int32_t* places;
    int n, Hq;
    int kv_splits, q_splits;      // CTAs that share a token's kv heads, query heads
};

constexpr int kAppendThreads = 256;
// Of K and V, loads of so many heads in flight: with one, two and four 4 x 8192
// tokens of 16-bit rows take 44, 41 and 70 us (registers).
constexpr int kAppendHeads = 2;

// How K and Q are rotated.
enum { kStay, kHalves, kInterleaved };

// A lane's eight channels of a row and, of halves, the other ones of their
// pairs. VEC: rows start on 16-byte boundaries and no piece is rotated in part;
// without it elements are loaded one by one.
template <typename T, bool VEC, int TURN>
struct Lane {
    Chunk<T, 8> own, other;

    __device__ __forceinline__ void load(const T* row, const RotaryDev& r, int d) {
        if (VEC) own.load(row + d);
        else own.load_each(row + d);
        if (TURN != kHalves || d >= r.R) return;
        const int half = r.R / 2;
        if constexpr (VEC) {
            other.load(row + (d < half ? d + half : d - half));
        } else {
            T e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = row[d + k < half ? d + k + half : d + k < r.R ? d + k - half : d + k];
            other.pack(e);
        }
    }
    // `c`, `s`: of this lane's channels (of halves), or pairs (interleaved); the first channel of a pair of
    // halves has its sine negated already.
    __device__ __forceinline__ void get(const RotaryDev& r, int d, const float (&c)[8], const float (&s)[8], float (&x)[8]) const {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = own.get(k);
        if constexpr (TURN != kStay) {
            if (d >= r.R) return;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (!VEC && d + k >= r.R) break;
                if (TURN == kHalves) {
                    x[k] = turned(x[k], other.get(k), c[k], s[k]);
                } else if (k % 2 == 0) {
                    const float a = x[k], z = x[k + 1];
                    x[k] = turned(a, z, c[k / 2], -s[k / 2]);
                    x[k + 1] = turned(z, a, c[k / 2], s[k / 2]);
                }
            }
        }
    }
};

// Cosines and sines as Lane::get takes them.
template <bool VEC, int TURN>
__device__ __forceinline__ void lane_turns(const RotaryDev& r, const int32_t* places, int64_t stride, int place, int d, float (&c)[8], float (&s)[8]) {
    if (TURN == kStay || d >= r.R) return;
    const int half = r.R / 2;
    if constexpr (TURN == kInterleaved) {
        if constexpr (VEC) {
            float cc[4], ss[4];
            load_turns<4>(r, places, stride, place, d / 2, cc, ss);
#pragma unroll
            for (int k = 0; k < 4; ++k) { c[k] = cc[k]; s[k] = ss[k]; }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float cc[1] = {0.f}, ss[1] = {0.f};
                if (d + 2 * k < r.R) load_turns<1>(r, places, stride, place, d / 2 + k, cc, ss);
                c[k] = cc[0];
                s[k] = ss[0];
            }
        }
    } else if constexpr (VEC) {
        load_turns<8>(r, places, stride, place, d < half ? d : d - half, c, s);
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = d < half ? -s[k] : s[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float cc[1] = {0.f}, ss[1] = {0.f};
            if (d + k < r.R) load_turns<1>(r, places, stride, place, d + k < half ? d + k : d + k - half, cc, ss);
            c[k] = cc[0];
            s[k] = d + k < half ? -ss[0] : ss[0];
        }
    }
}

// Scale of a group with the largest |x| `top` (a number).
__device__ __forceinline__ __half group_scale(float top) { return __float2half_rn(fminf(__fmul_rn(top, 1.f / 6.f), kMostScale)); }

// (0 with a scale of 0: a quotient keeps the sign of what it is of.)
__device__ __forceinline__ uint32_t group_codes(const float (&x)[8], float scale) {
    const float inverse = inverse_of(scale);
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = quotient(x[k], scale, inverse);
    return scale > 0.f ? to_codes(y) : 0u;
}

// grid.x: tokens of all sequences, so many rows of D / 8 lanes a CTA; grid.y:
// parts of the kv heads, then parts of the query heads.
template <typename T, bool VEC, int TURN>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(AppendParams p) {
    const CacheDev& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lanes = c.D / 8, rows = 32 / lanes;  // of a warp
    const int row_of_warp = lane / lanes, l = lane - row_of_warp * lanes, d = 8 * l;
    const int64_t token = (static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + warp) * rows + row_of_warp, tokens = static_cast<int64_t>(c.B) * p.n;
    const bool there = row_of_warp < rows && token < tokens;
    const int b = there ? static_cast<int>(token / p.n) : 0, i = there ? static_cast<int>(token - static_cast<int64_t>(b) * p.n) : 0;
    const int start = p.start[b], count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    const bool counted = there && i < count;
    float cs[8], sn[8];
    if (TURN != kStay && counted && d < p.r.R) {
        const int place = place_of(start, i);
        const int32_t* places = p.places ? p.places + token : nullptr;
        if (places_in(p.r, places, tokens, place)) {
            lane_turns<VEC, TURN>(p.r, places, tokens, place, d, cs, sn);
        } else {
            if (l == 0) q8::report(c.status, AKV_ERR_INVALID_ARGUMENT);
#pragma unroll
            for (int k = 0; k < 8; ++k) cs[k] = sn[k] = CUDART_NAN_F;
        }
    }
    if (static_cast<int>(blockIdx.y) >= p.kv_splits) {
        // Queries. (No lane waits for another here.)
        if (!there) return;
        const T* x = static_cast<const T*>(p.x[2]) + b * p.xB[2] + i * p.xT[2];
        T* out = static_cast<T*>(p.q_out) + token * p.Hq * c.D + d;
        for (int h0 = blockIdx.y - p.kv_splits; h0 < p.Hq; h0 += 2 * p.q_splits) {
            Lane<T, VEC, TURN> v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (counted && h0 + j * p.q_splits < p.Hq) v[j].load(x + (h0 + j * p.q_splits) * p.xH[2], p.r, d);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int h = h0 + j * p.q_splits;
                if (h >= p.Hq) break;
                float y[8];
                if (counted) {
                    v[j].get(p.r, d, cs, sn, y);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = 0.f;
                }
                Chunk<T, 8> o;
                o.set(y);
                o.store(out + static_cast<int64_t>(h) * c.D);
            }
        }
        return;
    }
    if (there && i == 0 && l == 0 && blockIdx.y == 0 && count > 0 && (start < 0 || static_cast<int64_t>(start) + count > c.T))
        q8::report(c.status, AKV_ERR_INVALID_ARGUMENT);
    const bool kept = counted && start >= 0 && start < c.T && i < c.T - start;
    int row = 0;
    const int phys = kept ? page_of(c, b, start + i, row) : -1;
    if (!__any_sync(0xFFFFFFFFu, phys >= 0)) return;
    const bool store = phys >= 0;
    const uint32_t row_mask = (lanes == 32 ? 0xFFFFFFFFu : (1u << lanes) - 1) << (row_of_warp * lanes & 31);
    const T* xk = static_cast<const T*>(p.x[0]) + b * p.xB[0] + i * p.xT[0];
    const T* xv = static_cast<const T*>(p.x[1]) + b * p.xB[1] + i * p.xT[1];
    for (int h0 = blockIdx.y; h0 < c.H; h0 += 2 * p.kv_splits) {
        Lane<T, VEC, TURN> k2[2];
        Lane<T, VEC, kStay> v2[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = h0 + j * p.kv_splits;
            if (!store || h >= c.H) continue;
            k2[j].load(xk + h * p.xH[0], p.r, d);
            v2[j].load(xv + h * p.xH[1], p.r, d);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = h0 + j * p.kv_splits;
            if (h >= c.H) break;
            float x[2][8];
            uint32_t top[2] = {0, 0};
            if (store) {
                k2[j].get(p.r, d, cs, sn, x[0]);
                v2[j].get(p.r, d, cs, sn, x[1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    top[0] = max(top[0], q8::abs_bits(x[0][e]));
                    top[1] = max(top[1], q8::abs_bits(x[1][e]));
                }
            }
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {
                top[0] = max(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], o));
                top[1] = max(top[1], __shfl_xor_sync(0xFFFFFFFFu, top[1], o));
            }
            const uint32_t inf = 0x7F800000u;
            const bool bad = __ballot_sync(0xFFFFFFFFu, top[0] >= inf || top[1] >= inf) & row_mask;
            if (!store) continue;
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                const SideDev& s = side ? c.v : c.k;
                const bool none = side ? top[1] >= inf : bad;
                const __half scale = none ? __ushort_as_half(side ? 0 : 0x7FFF) : group_scale(__uint_as_float(top[side]));
                const uint32_t w = none ? 0u : group_codes(x[side], __half2float(scale));
                *reinterpret_cast<uint32_t*>(s.codes + code_offset(s, b, h, phys, row) + 4 * l) = w;
                if ((l & 3) == 0) s.scales[scale_offset(s, b, h, phys, row) + (l >> 2) * s.cG] = scale;
            }
        }
    }
}

// ------------------------------------------------- pairs of chunks a lane
//
// The form that a model's prompts and steps take: 16-byte rows, pairs of
// halves (or none), and halves that hold whole groups. A lane has two chunks of eight
// channels, of rotated ones the two halves of eight pairs, so that nothing is
// loaded twice, and two fp32 operations go in one instruction.

__device__ __forceinline__ uint64_t pack2f(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float2 unpack2f(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t fma2f(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2f(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// The sums of products have to be rounded by themselves. As pairs the compiler
// makes a multiplication and an addition one operation (also where they are
// written as two), so additions are done one by one.
__device__ __forceinline__ uint64_t sum2f(uint64_t a, uint64_t b, float sign) {
    const float2 x = unpack2f(a), y = unpack2f(b);
    return sign < 0.f ? pack2f(__fsub_rn(x.x, y.x), __fsub_rn(x.y, y.y)) : pack2f(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
// The largest |x|, a NaN if one is.
__device__ __forceinline__ float largest_of(const uint64_t (&x)[4]) {
    float top[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2f(x[k]);
        top[0] = max_nan(top[0], fabsf(f.x));
        top[1] = max_nan(top[1], fabsf(f.y));
    }
    return max_nan(top[0], top[1]);
}

// Eight channels as four pairs of neighbours.
template <typename T>
__device__ __forceinline__ void chunk_values(const Chunk<T, 8>& v, uint64_t (&x)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = pack2f(v.get(2 * k), v.get(2 * k + 1));
}

// Codes of a chunk, given its group's scale.
__device__ __forceinline__ uint32_t chunk_codes(const uint64_t (&x)[4], float scale) {
    const float inverse = inverse_of(scale);
    const uint64_t inv = pack2f(inverse, inverse), neg = pack2f(-scale, -scale);
    float y[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint64_t q = mul2f(x[k], inv);  // see quotient()
        const float2 f = unpack2f(fma2f(fma2f(q, neg, x[k]), inv, q));
        y[2 * k] = f.x;
        y[2 * k + 1] = f.y;
    }
    return scale > 0.f ? to_codes(y) : 0u;
}

// Grid as of append_kernel, with rows of D / 16 lanes. QUERIES: with parts for
// the query heads. Two CTAs an SM of fp32 rows (with the registers of one 75 us
// for 4 x 8192 tokens, so 55).
template <typename T, bool TURN, bool QUERIES>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 4 || QUERIES ? 2 : 3) append_pairs_kernel(AppendParams p) {
    const CacheDev& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lanes = c.D / 16, rows = 32 / lanes;  // of a warp
    const int row_of_warp = lane / lanes, u = lane - row_of_warp * lanes;
    const int64_t token = (static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + warp) * rows + row_of_warp, tokens = static_cast<int64_t>(c.B) * p.n;
    const bool there = row_of_warp < rows && token < tokens;
    const int b = there ? static_cast<int>(token / p.n) : 0, i = there ? static_cast<int>(token - static_cast<int64_t>(b) * p.n) : 0;
    const int start = p.start[b], count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    const bool counted = there && i < count;
    // The lane's chunks: of the rotated channels, then of the others, half of them apart.
    const int R = TURN ? p.r.R : 0;
    const bool turn = TURN && 16 * u < R;
    const int d0 = turn ? 8 * u : R + 8 * (u - R / 16), d1 = d0 + (turn ? R / 2 : (c.D - R) / 2);
    uint64_t cs[4], sn[4];
    if (turn && counted) {
        const int place = place_of(start, i);
        const int32_t* places = p.places ? p.places + token : nullptr;
        float cc[8], ss[8];
        if (places_in(p.r, places, tokens, place)) {
            load_turns<8>(p.r, places, tokens, place, d0, cc, ss);
        } else {
            if (u == 0) q8::report(c.status, AKV_ERR_INVALID_ARGUMENT);
#pragma unroll
            for (int k = 0; k < 8; ++k) cc[k] = ss[k] = CUDART_NAN_F;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cs[k] = pack2f(cc[2 * k], cc[2 * k + 1]);
            sn[k] = pack2f(ss[2 * k], ss[2 * k + 1]);
        }
    }
    auto rotate = [&](uint64_t (&x)[4], uint64_t (&z)[4]) {
        if constexpr (TURN) {
            if (!turn) return;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint64_t e = sum2f(mul2f(x[k], cs[k]), mul2f(z[k], sn[k]), -1.f), f = sum2f(mul2f(z[k], cs[k]), mul2f(x[k], sn[k]), 1.f);
                x[k] = e;
                z[k] = f;
            }
        }
    };
    if (QUERIES && static_cast<int>(blockIdx.y) >= p.kv_splits) {
        // Queries. (No lane waits for another here.)
        if (!there) return;
        const T* x = static_cast<const T*>(p.x[2]) + b * p.xB[2] + i * p.xT[2];
        T* out = static_cast<T*>(p.q_out) + token * p.Hq * c.D;
        for (int h0 = blockIdx.y - p.kv_splits; h0 < p.Hq; h0 += kRotateHeads * p.q_splits) {
            Chunk<T, 8> v[kRotateHeads][2];
#pragma unroll
            for (int j = 0; j < kRotateHeads; ++j) {
                const int h = h0 + j * p.q_splits;
                if (!counted || h >= p.Hq) break;
                v[j][0].load(x + h * p.xH[2] + d0);
                v[j][1].load(x + h * p.xH[2] + d1);
            }
#pragma unroll
            for (int j = 0; j < kRotateHeads; ++j) {
                const int h = h0 + j * p.q_splits;
                if (h >= p.Hq) break;
                Chunk<T, 8> o[2];
                if (counted) {
                    uint64_t y[2][4];
                    chunk_values(v[j][0], y[0]);
                    chunk_values(v[j][1], y[1]);
                    rotate(y[0], y[1]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float f[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float2 g = unpack2f(y[e][k]);
                            f[2 * k] = g.x;
                            f[2 * k + 1] = g.y;
                        }
                        o[e].set(f);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int k = 0; k < Chunk<T, 8>::kWords; ++k) o[e].w[k] = 0;
                }
                o[0].store(out + static_cast<int64_t>(h) * c.D + d0);
                o[1].store(out + static_cast<int64_t>(h) * c.D + d1);
            }
        }
        return;
    }
    if (there && i == 0 && u == 0 && blockIdx.y == 0 && count > 0 && (start < 0 || static_cast<int64_t>(start) + count > c.T))
        q8::report(c.status, AKV_ERR_INVALID_ARGUMENT);
    const bool kept = counted && start >= 0 && start < c.T && i < c.T - start;
    int row = 0;
    const int phys = kept ? page_of(c, b, start + i, row) : -1;
    if (!__any_sync(0xFFFFFFFFu, phys >= 0)) return;
    const bool store = phys >= 0;
    const uint32_t row_mask = (lanes == 32 ? 0xFFFFFFFFu : (1u << lanes) - 1) << (row_of_warp * lanes & 31);
    // Where the lane's first chunk of the next head is, stepped from head to
    // head: multiplied out for each, offsets were a quarter of the instructions
    // (51 against 43 us for 4 x 8192 tokens of 8 heads).
    const int h_first = blockIdx.y;
    const T* in[2];
    uint8_t* codes[2];
    __half* scales[2];
    const int apart = d1 - d0;
    int64_t in_step[2], code_step[2], scale_step[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const SideDev& s = side ? c.v : c.k;
        in_step[side] = p.kv_splits * p.xH[side];
        code_step[side] = p.kv_splits * s.sH;
        scale_step[side] = p.kv_splits * s.cH;
        in[side] = static_cast<const T*>(p.x[side]) + b * p.xB[side] + i * p.xT[side] + h_first * p.xH[side] + d0;
        codes[side] = s.codes + code_offset(s, b, h_first, phys, row) + d0 / 2;
        scales[side] = s.scales + scale_offset(s, b, h_first, phys, row) + d0 / AKV_Q4_GROUP * s.cG;
    }
    for (int h0 = blockIdx.y; h0 < c.H; h0 += kAppendHeads * p.kv_splits) {
        Chunk<T, 8> v[kAppendHeads][2][2];  // [head][side][chunk]
#pragma unroll
        for (int j = 0; j < kAppendHeads; ++j) {
            const int h = h0 + j * p.kv_splits;
#pragma unroll
            for (int side = 0; side < 2; ++side)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    v[j][side][e].clear();  // a lane that stores nothing goes along with zeros
                    if (store && h < c.H) v[j][side][e].load(in[side] + e * apart);
                }
            in[0] += in_step[0];
            in[1] += in_step[1];
        }
#pragma unroll
        for (int j = 0; j < kAppendHeads; ++j) {
            const int h = h0 + j * p.kv_splits;
            if (h >= c.H) break;
            bool mine = true;  // of this lane's groups, whether all are numbers
            // V, then K, which has to know of V.
#pragma unroll
            for (int side = 1; side >= 0; --side) {
                const SideDev& s = side ? c.v : c.k;
                uint64_t x[2][4];
                float top[2];
                chunk_values(v[j][side][0], x[0]);
                chunk_values(v[j][side][1], x[1]);
                if (side == 0) rotate(x[0], x[1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) top[e] = side == 0 || sizeof(T) == 4 ? largest_of(x[e]) : v[j][side][e].largest();
#pragma unroll
                for (int o = 1; o <= 2; o <<= 1) {
                    top[0] = max_nan(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], o));
                    top[1] = max_nan(top[1], __shfl_xor_sync(0xFFFFFFFFu, top[1], o));
                }
                const bool fine[2] = {top[0] < CUDART_INF_F, top[1] < CUDART_INF_F};
                mine = mine && fine[0] && fine[1];
                bool bad = false;
                if (side == 0) bad = __ballot_sync(0xFFFFFFFFu, !mine) & row_mask;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool none = side ? !fine[e] : bad;
                    const __half scale = none ? __ushort_as_half(side ? 0 : 0x7FFF) : group_scale(top[e]);
                    const uint32_t w = none ? 0u : chunk_codes(x[e], __half2float(scale));
                    if (store) *reinterpret_cast<uint32_t*>(codes[side] + e * apart / 2) = w;
                    if (store && (u & 3) == 0) scales[side][e * apart / AKV_Q4_GROUP * s.cG] = scale;
                }
                codes[side] += code_step[side];
                scales[side] += scale_step[side];
            }
        }
    }
}

struct RestoreParams {
    CacheDev c;
    void* out[2];
    const int32_t* start;
    int n;
};

// One thread per sixteen channels (eight bytes of codes, 32 or 64 of values), in
// the order of the output, so that stores are whole lines; grid.y: sequence x side.
template <typename T>
__global__ void __launch_bounds__(256) restore_kernel(RestoreParams p) {
    const CacheDev& c = p.c;
    const int b = blockIdx.y >> 1, side = blockIdx.y & 1;
    const SideDev& s = side ? c.v : c.k;
    const unsigned per_row = c.D / 16, per_token = per_row * c.H;
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= per_token * p.n) return;
    const unsigned ti = i / per_token, rest = i - ti * per_token;
    const int h = rest / per_row, l = rest - h * per_row;
    q8::wait_for_previous_kernel();
    const int64_t t = static_cast<int64_t>(ti) + (p.start ? p.start[b] : 0);
    int row = 0;
    const int phys = t >= 0 && t < c.T ? page_of(c, b, static_cast<int>(t), row) : -1;
    uint2 w = make_uint2(0, 0);
    __half scale = __float2half_rn(0.f);
    if (phys >= 0) {
        w = *reinterpret_cast<const uint2*>(s.codes + code_offset(s, b, h, phys, row) + 8 * l);
        scale = s.scales[scale_offset(s, b, h, phys, row) + (l >> 1) * s.cG];
    }
    const __half2 both = __half2half2(scale);
    T* out = static_cast<T*>(p.out[side]) + (static_cast<int64_t>(b) * p.n * per_token + i) * 16;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        uint32_t v[4];
        codes_to_half(e ? w.y : w.x, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = mul2(v[k], *reinterpret_cast<const uint32_t*>(&both));
        Chunk<T, 8> o;
        if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
            for (int k = 0; k < 4; ++k) o.w[k] = v[k];
        } else {
            float x[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[k]));
                x[2 * k] = f.x;
                x[2 * k + 1] = f.y;
            }
            o.set(x);
        }
        o.store(out + 8 * e);
    }
}

}  // namespace q4
}  // namespace akv
