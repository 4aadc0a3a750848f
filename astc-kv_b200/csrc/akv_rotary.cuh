// Rotary positions: the kernel that rotates the heads of tokens, and what an
// append to the 4-bit cache shares with it.
//
// A pair (x1, x2) at angle a becomes (x1 cos a - x2 sin a, x2 cos a + x1 sin a).
// Cosines and sines are read from a table, made once in 64 bits: a fp32 angle
// of position 131071 is off by 2^-8, and a polynomial for sines would cost
// more than the 8 bytes a pair, which all heads of a token share. Products and sums
// are rounded one by one (no fused multiply-add), so that every call that
// rotates a value gets the same bits.
#pragma once
#include <math_constants.h>

#include "../../include/akv_rotary.h"
#include "akv_q8_common.cuh"

namespace akv {

struct RotaryDev {
    const float* table;
    int positions, R, axes;
    uint32_t used;           // axes that a pair takes
    bool whole_rows;         // rows of the table start on 16-byte boundaries
    uint8_t axis[128];
};

inline RotaryDev to_dev(const AkvRotary& r) {
    RotaryDev d;
    d.table = r.table_dev;
    d.positions = r.positions; d.R = r.rotary_dim; d.axes = r.axes;
    d.used = 0;
    d.whole_rows = r.rotary_dim % 4 == 0;
    for (int i = 0; i < r.rotary_dim / 2; ++i) {
        d.axis[i] = r.axis[i];
        d.used |= 1u << r.axis[i];
    }
    return d;
}

inline int check_rotary(const AkvRotary& r, int head_dim) {
    if (!r.table_dev || reinterpret_cast<uintptr_t>(r.table_dev) % 16 || r.positions <= 0) return AKV_ERR_INVALID_ARGUMENT;
    if (r.rotary_dim <= 0 || r.rotary_dim % 2 || r.rotary_dim > head_dim || r.axes <= 0) return AKV_ERR_INVALID_ARGUMENT;
    if (r.rotary_dim > 256 || r.axes > AKV_ROTARY_MAX_AXES) return AKV_ERR_UNSUPPORTED;
    for (int i = 0; i < r.rotary_dim / 2; ++i)
        if (r.axis[i] >= r.axes) return AKV_ERR_INVALID_ARGUMENT;
    return AKV_OK;
}

// Whether a token's positions are in the table: of axis a the one at
// places[a * stride], or `place` on every axis without places.
__device__ __forceinline__ bool places_in(const RotaryDev& r, const int32_t* places, int64_t stride, int place) {
    if (!places) return static_cast<unsigned>(place) < static_cast<unsigned>(r.positions);
    bool in = true;
    for (int a = 0; a < r.axes; ++a)
        if (r.used >> a & 1) in = in && static_cast<unsigned>(__ldg(places + a * stride)) < static_cast<unsigned>(r.positions);
    return in;
}

// Cosines and sines of pairs first .. first + N - 1 of a token (see places_in,
// which has to be true). N is 1, or first is a multiple of 4.
template <int N>
__device__ __forceinline__ void load_turns(const RotaryDev& r, const int32_t* places, int64_t stride, int place, int first, float (&c)[N], float (&s)[N]) {
    const int64_t row = r.R;  // floats
    if (N >= 4 && r.whole_rows && (r.axes == 1 || !places)) {
        const float4* at = reinterpret_cast<const float4*>(r.table + (places ? __ldg(places) : place) * row + 2 * first);
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            const float4 v = __ldg(at + k);
            c[2 * k] = v.x; s[2 * k] = v.y;
            c[N > 1 ? 2 * k + 1 : 0] = v.z; s[N > 1 ? 2 * k + 1 : 0] = v.w;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int p = places ? __ldg(places + r.axis[first + k] * stride) : place;
        const float2 v = __ldg(reinterpret_cast<const float2*>(r.table + p * row) + first + k);
        c[k] = v.x;
        s[k] = v.y;
    }
}

// x cos + other sin: the first of a pair gives -sin.
__device__ __forceinline__ float turned(float x, float other, float c, float s) { return __fadd_rn(__fmul_rn(x, c), __fmul_rn(other, s)); }

// N consecutive elements as they are in memory.
template <typename T, int N>
struct Chunk {
    static constexpr int kBytes = N * sizeof(T), kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];

    // Aligned to its size, at most 16 bytes.
    __device__ __forceinline__ void load(const T* at) {
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int k = 0; k < kBytes / 16; ++k) {
                const uint4 v = *(reinterpret_cast<const uint4*>(at) + k);
                w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
            }
        } else if constexpr (kBytes == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            w[0] = v.x; w[1] = v.y;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(at);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(at);
        }
    }
    __device__ __forceinline__ void store(T* at) const {
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int k = 0; k < kBytes / 16; ++k) *(reinterpret_cast<uint4*>(at) + k) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        } else if constexpr (kBytes == 8) {
            *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
        } else if constexpr (kBytes == 4) {
            *reinterpret_cast<uint32_t*>(at) = w[0];
        } else {
            *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(w[0]);
        }
    }
    // Element by element, wherever it starts.
    __device__ __forceinline__ void load_each(const T* at) {
        T e[N];
#pragma unroll
        for (int k = 0; k < N; ++k) e[k] = at[k];
        pack(e);
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const uint32_t v = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu;
            if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(v << 16);
            else return __half2float(__ushort_as_half(static_cast<uint16_t>(v)));
        }
    }
    __device__ __forceinline__ void set(const float (&x)[N]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < N; ++k) w[k] = __float_as_uint(x[k]);
        } else if constexpr (N == 1) {
            w[0] = q8::pack2<T>(x[0], x[0]) & 0xFFFFu;
        } else {
#pragma unroll
            for (int k = 0; k < N / 2; ++k) w[k] = q8::pack2<T>(x[2 * k], x[2 * k + 1]);
        }
    }
    __device__ __forceinline__ void pack(const T (&e)[N]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < N; ++k) w[k] = *reinterpret_cast<const uint32_t*>(&e[k]);
        } else {
            const uint16_t* u = reinterpret_cast<const uint16_t*>(e);
#pragma unroll
            for (int k = 0; k < kWords; ++k) w[k] = u[2 * k] | (N > 1 ? static_cast<uint32_t>(u[N > 1 ? 2 * k + 1 : 0]) << 16 : 0u);
        }
    }
};

struct RotateParams {
    RotaryDev r;
    int B, n, H, D;
    int splits;                // threads that share a token's heads
    bool inverse;
    const void* x;
    void* out;
    int64_t xB, xT, xH, oB, oT, oH;  // elements
    const int32_t* places;
    int32_t* status;
};

constexpr int kRotateThreads = 256;
constexpr int kRotateHeads = 4;  // loads of so many heads in flight

// A thread has a unit of N pairs, or 2 N channels that stay, of one token, and
// every splits-th head: cosines and sines are read once for them all. Since it reads
// what it writes and nothing else, out may be x.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(RotateParams p) {
    const unsigned units = (p.D + 2 * N - 1) / (2 * N);
    const unsigned i = blockIdx.x * static_cast<unsigned>(kRotateThreads) + threadIdx.x, rest = i / units, u = i - rest * units;
    const unsigned token = rest / p.splits, split = rest - token * p.splits;
    if (token >= static_cast<unsigned>(p.B) * p.n) return;
    const int b = token / p.n, t = token - b * p.n;
    const bool turn = static_cast<int>(2 * N * u) < p.r.R;
    const int at0 = turn && !INTER ? N * u : 2 * N * u, at1 = turn && !INTER ? at0 + p.r.R / 2 : at0 + N;
    const bool second = N > 1 || at1 < p.D;
    const T* x = static_cast<const T*>(p.x) + b * p.xB + t * p.xT;
    T* out = static_cast<T*>(p.out) + b * p.oB + t * p.oT;
    float c[N], s[N];
    if (turn) {
        const int32_t* places = p.places + token;
        const int64_t stride = static_cast<int64_t>(p.B) * p.n;
        if (places_in(p.r, places, stride, 0)) {
            load_turns<N>(p.r, places, stride, 0, N * u, c, s);
            if (p.inverse) {
#pragma unroll
                for (int k = 0; k < N; ++k) s[k] = -s[k];
            }
        } else {
            if (u == 0) q8::report(p.status, AKV_ERR_INVALID_ARGUMENT);
#pragma unroll
            for (int k = 0; k < N; ++k) c[k] = s[k] = CUDART_NAN_F;
        }
    }
    for (int h0 = split; h0 < p.H; h0 += kRotateHeads * p.splits) {
        Chunk<T, N> v[kRotateHeads][2];
#pragma unroll
        for (int j = 0; j < kRotateHeads; ++j) {
            const int h = h0 + j * p.splits;
            if (h >= p.H) break;
            v[j][0].load(x + h * p.xH + at0);
            if (second) v[j][1].load(x + h * p.xH + at1);
        }
#pragma unroll
        for (int j = 0; j < kRotateHeads; ++j) {
            const int h = h0 + j * p.splits;
            if (h >= p.H) break;
            if (turn) {
                float y1[N], y2[N];
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const float a = INTER ? (2 * k < N ? v[j][0].get(2 * k % N) : v[j][1].get(2 * k % N)) : v[j][0].get(k);
                    const float z = !INTER ? v[j][1].get(k) : N == 1 ? v[j][1].get(0) : 2 * k < N ? v[j][0].get((2 * k + 1) % N) : v[j][1].get((2 * k + 1) % N);
                    const float e = turned(a, z, c[k], -s[k]), f = turned(z, a, c[k], s[k]);
                    if (!INTER || N == 1) {
                        y1[k] = e;
                        y2[k] = f;
                    } else if (2 * k < N) {
                        y1[2 * k % N] = e;
                        y1[(2 * k + 1) % N] = f;
                    } else {
                        y2[2 * k % N] = e;
                        y2[(2 * k + 1) % N] = f;
                    }
                }
                v[j][0].set(y1);
                v[j][1].set(y2);
            }
            v[j][0].store(out + h * p.oH + at0);
            if (second) v[j][1].store(out + h * p.oH + at1);
        }
    }
}

}  // namespace akv
