// Loads of the 4-bit cache's attention kernels.
#pragma once
#include "akv_q4_attend.cuh"

namespace akv {
namespace q4 {

// Four scales.
__device__ __forceinline__ uint2 load_scales(const __half* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
// NWORDS words, 4 to 16 bytes.
template <int NWORDS>
__device__ __forceinline__ void load_words(uint32_t (&w)[NWORDS], const uint8_t* p) {
    if constexpr (NWORDS == 4) {
        const uint4 v = q8::load_stream(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (NWORDS == 2) {
        const uint2 v = q8::load_stream8(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
    }
}

}  // namespace q4
}  // namespace akv
