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
    int wait_tries;     // of a wait in the tcgen05 kernel
};

// Host launchers of the step kernel, one translation unit each (the kernel has
// many instances; they compile side by side). nt: groups of eight rows per CTA, 1 or 2.
int launch_step_dense(const Q4Params& p, int nt, cudaStream_t s);    // see the kernel's DENSE
int launch_step_strided(const Q4Params& p, int nt, cudaStream_t s);

}  // namespace q4
}  // namespace akv
