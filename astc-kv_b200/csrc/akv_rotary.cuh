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
#include <climits>

#include <math_constants.h>

#include <initializer_list>

#include "../../include/akv_rotary.h"
#include "akv_q8_common.cuh"

namespace akv {

struct RotaryDev {
    const float* table;
    int positions, R, axes;
    uint32_t used;           // axes that a pair takes
    uint32_t alike;          // bit i: pairs 4i to 4i + 3 take one axis
    bool whole_rows;         // rows of the table start on 16-byte boundaries
    uint8_t axis[128];
};

inline RotaryDev to_dev(const AkvRotary& r) {
    RotaryDev d;
    d.table = r.table_dev;
    d.positions = r.positions; d.R = r.rotary_dim; d.axes = r.axes;
    d.used = 0;
    d.alike = ~0u;
    d.whole_rows = r.rotary_dim % 4 == 0;
    for (int i = 0; i < r.rotary_dim / 2; ++i) {
        d.axis[i] = r.axis[i];
        d.used |= 1u << r.axis[i];
        if (i % 4 && r.axis[i] != r.axis[i - 1]) d.alike &= ~(1u << i / 4);
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
    if constexpr (N >= 4) {
        constexpr uint32_t all = (1u << N / 4) - 1;
        const int axis = r.axis[first];
        if (r.whole_rows && (!places || ((r.alike >> first / 4 & all) == all && axis == r.axis[first + N - 4]))) {
            const float4* at = reinterpret_cast<const float4*>(r.table + (places ? __ldg(places + axis * stride) : place) * row + 2 * first);
#pragma unroll
            for (int k = 0; k < N / 2; ++k) {
                const float4 v = __ldg(at + k);
                c[2 * k] = v.x; s[2 * k] = v.y;
                c[2 * k + 1] = v.z; s[2 * k + 1] = v.w;
            }
            return;
        }
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

__device__ __forceinline__ __half low_of(__half2 v) { return __low2half(v); }
__device__ __forceinline__ __half high_of(__half2 v) { return __high2half(v); }
__device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 v) { return __low2bfloat16(v); }
__device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 v) { return __high2bfloat16(v); }

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
                // (Volatile, so that all of a round's loads stay ahead of its arithmetic; not from the
                // read-only path: out may be x.)
                uint4 v;
                asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(reinterpret_cast<const uint4*>(at) + k) : "memory");
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
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = 0;
    }
    // The largest |element| of 16-bit ones, a NaN if one is.
    __device__ __forceinline__ float largest() const {
        if constexpr (sizeof(T) == 2) {
            using T2 = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>;
            T2 m = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
            for (int k = 1; k < kWords; ++k) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2*>(&w[k])));
            const T top = __hmax_nan(low_of(m), high_of(m));
            return static_cast<float>(top);
        } else {
            return 0.f;
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
    const int32_t* places;     // or NULL: the tokens' places in a cache, start[b] + i
    const int32_t* start;
    const int32_t* counts;     // tokens of each sequence, zeros past them; or NULL
    int32_t* status;
};

// Token i of a sequence that begins at `start`. (A start outside a cache may be none of the table either.)
__device__ __forceinline__ int place_of(int start, int i) { return static_cast<int>(min(static_cast<int64_t>(start) + i, static_cast<int64_t>(INT_MAX))); }

constexpr int kRotateThreads = 256;
constexpr int kRotateHeads = 4;  // loads of so many heads in flight

// A thread has a unit of N pairs, or 2 N channels that stay, of one token, and
// every splits-th head: cosines and sines are read once for them all. Since it reads
// what it writes and nothing else, out may be x.
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(RotateParams p) {
    constexpr bool ONE = INTER && sizeof(Chunk<T, 2 * N>) == 16;  // both pieces are 16 bytes in a row
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
    const bool counted = !p.counts || t < p.counts[b];
    if (turn && counted) {
        const int32_t* places = p.places ? p.places + token : nullptr;
        const int64_t stride = static_cast<int64_t>(p.B) * p.n;
        const int place = p.start ? place_of(p.start[b], t) : 0;
        if (places_in(p.r, places, stride, place)) {
            load_turns<N>(p.r, places, stride, place, N * u, c, s);
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
            v[j][0].clear();
            v[j][1].clear();
            if (!counted) continue;
            if constexpr (ONE) {
                Chunk<T, 2 * N> both;
                both.load(x + h * p.xH + at0);
#pragma unroll
                for (int k = 0; k < Chunk<T, N>::kWords; ++k) {
                    v[j][0].w[k] = both.w[k];
                    v[j][1].w[k] = both.w[k + Chunk<T, N>::kWords];
                }
            } else {
                v[j][0].load(x + h * p.xH + at0);
                if (second) v[j][1].load(x + h * p.xH + at1);
            }
        }
#pragma unroll
        for (int j = 0; j < kRotateHeads; ++j) {
            const int h = h0 + j * p.splits;
            if (h >= p.H) break;
            if (turn && counted) {
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
            if constexpr (ONE) {
                Chunk<T, 2 * N> both;
#pragma unroll
                for (int k = 0; k < Chunk<T, N>::kWords; ++k) {
                    both.w[k] = v[j][0].w[k];
                    both.w[k + Chunk<T, N>::kWords] = v[j][1].w[k];
                }
                both.store(out + h * p.oH + at0);
            } else {
                v[j][0].store(out + h * p.oH + at0);
                if (second) v[j][1].store(out + h * p.oH + at1);
            }
        }
    }
}

// How wide rotate_kernel's pieces may be: 8 pairs (16 bytes of either half), 4
// pairs, else one; for the addresses and strides (bytes) of its rows.
inline int rotate_width(const RotateParams& p, bool interleaved, int64_t elem) {
    const auto aligned = [&](int64_t bytes) {
        bool a = reinterpret_cast<uintptr_t>(p.x) % bytes == 0 && reinterpret_cast<uintptr_t>(p.out) % bytes == 0;
        for (const int64_t st : {p.xB, p.xT, p.xH, p.oB, p.oT, p.oH}) a = a && st * elem % bytes == 0;
        return a;
    };
    if (elem == 2 && !interleaved && p.r.R % 16 == 0 && p.D % 16 == 0 && aligned(16)) return 8;
    return p.r.R % 8 == 0 && p.D % 8 == 0 && aligned(interleaved ? 16 : 4 * elem) ? 4 : 1;
}

// Threads that share a token's heads. Eight heads a thread (4 x 8191 tokens, 40
// heads, D 128, bf16: 109 us, with four 121, with twenty 111), twenty where
// positions have several axes and a thread takes longer to begin (113 us against
// 118; both with 40 heads, no other number was measured), fewer where that leaves SMs with few threads (2 x 4097 tokens, 16 heads, D 72:
// 10.3 us, with 2048 threads an SM asked for 12.4). 0 where the grid would be too large.
inline int rotate_splits(const RotateParams& p, int N) {
    const int64_t units = static_cast<int64_t>(p.B) * p.n * ((p.D + 2 * N - 1) / (2 * N)), few = 148 * 640;
    const int64_t want = (few + units - 1) / units, heads = p.r.axes > 1 && p.places ? 20 : 8;
    int64_t splits = (p.H + heads - 1) / heads;
    if (splits < want) splits = want < p.H ? want : p.H;
    if (units * splits > 0x7FFFFF00) splits = 1;
    return units * splits > 0x7FFFFF00 ? 0 : static_cast<int>(splits);
}

// Whether one launch holds them.
inline bool rotate_fits(const RotateParams& p, int dtype, bool interleaved) {
    return rotate_splits(p, rotate_width(p, interleaved, dtype == AKV_Q_F32 ? 4 : 2)) > 0;
}

// Launches rotate_kernel; dtype AKV_Q_*. Defined in akv_rotary.cu.
int launch_rotate(RotateParams p, int dtype, bool interleaved, cudaStream_t s);

}  // namespace akv
