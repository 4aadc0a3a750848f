// Attention over the 4-bit KV cache: parameters shared by its kernels.
//
// The division of the work, the partials and their combination do not depend
// on what the cache holds: they are those of the 8-bit cache's step and combine kernels.
#pragma once
#include "akv_q4_common.cuh"
#include "akv_q8_step.cuh"

namespace akv {
namespace q4 {

struct Q4Params {
    q8::AttnParams a;   // of a.c only B, H, D, T and status are set
    CacheDev c;
    bool long_sums;     // of a CTA of the step kernel, see kStepLong
    int wait_tries;     // of a wait in the tcgen05 kernel
};

// Tokens that a CTA of the step kernel with a 16-bit output may go through in one sum, or
// puts its sum by after: the tensor cores truncate as they add, so a sum over n tokens
// comes out about 6e-9 n too small, which an output's rounding (2^-11, fp16; 2^-8,
// bf16) has to cover. Of these tokens a warp adds up a quarter. (With every sum put
// by after 16384 tokens 32 sequences of 32768, 32/8 heads of 128 channels, bf16, took
// 242 us where they take 232, although none of their sums is that long.)
constexpr int kStepLong = 65536, kStepLongBf16 = 8 * kStepLong;

// Host launchers of the step kernel, one translation unit each (the kernel has
// many instances; they compile side by side). nt: groups of eight rows per CTA, 1 or 2.
int launch_step_dense(const Q4Params& p, int nt, cudaStream_t s);    // see the kernel's DENSE
int launch_step_strided(const Q4Params& p, int nt, cudaStream_t s);

}  // namespace q4
}  // namespace akv
