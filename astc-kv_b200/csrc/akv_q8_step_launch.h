// Host launchers of the step kernel, one translation unit per code format (the
// kernel has many instances; they compile side by side).
#pragma once
#include "akv_q8_attend.cuh"

namespace akv {
namespace q8 {

constexpr int kStepCluster = 8;   // CTAs of a cluster at most
constexpr int kStepWarps = 4;     // warps of a CTA, a tile of 16 tokens each

inline int launched() { return cudaPeekAtLastError() == cudaSuccess ? AKV_OK : (cudaGetLastError(), AKV_ERR_CUDA); }

// nt: groups of eight rows per CTA, 1 or 2.
int launch_step_int8(const AttnParams& p, int nt, cudaStream_t s);
int launch_step_e4m3(const AttnParams& p, int nt, cudaStream_t s);

}  // namespace q8
}  // namespace akv
