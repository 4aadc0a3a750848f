// Template dispatch of the step kernel, included by akv_q8_step_*.cu.
#pragma once
#include "akv_q8_step.cuh"

namespace akv {
namespace q8 {
namespace {

template <int FMT, int DP, int NT, bool PLO, bool QLO, bool TWIN>
int launch_step(const AttnParams& p, cudaStream_t s) {
    if constexpr (NT == 1) {
        if (p.share_ctas < 0) {
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = static_cast<unsigned>(-p.share_ctas);
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(static_cast<unsigned>(p.c.B) * p.c.H * static_cast<unsigned>(-p.share_ctas));
            cfg.blockDim = dim3(kStepThreads);
            cfg.stream = s;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            return cudaLaunchKernelEx(&cfg, step_kernel<FMT, DP, 1, PLO, QLO, TWIN, true>, p) == cudaSuccess
                       ? AKV_OK : (cudaGetLastError(), AKV_ERR_CUDA);
        }
    }
    step_kernel<FMT, DP, NT, PLO, QLO, TWIN, false><<<p.share_ctas, kStepThreads, 0, s>>>(p);
    return launched();
}

template <int FMT, int DP, int NT>
int launch_step(const AttnParams& p, cudaStream_t s) {
    const bool plo = p.out_dtype == AKV_Q_F32, qlo = p.q_dtype == AKV_Q_F32;
    if constexpr (NT == 1) {
        if (plo && p.R <= 4) return qlo ? launch_step<FMT, DP, 1, true, true, true>(p, s) : launch_step<FMT, DP, 1, true, false, true>(p, s);
    }
    if (plo) return qlo ? launch_step<FMT, DP, NT, true, true, false>(p, s) : launch_step<FMT, DP, NT, true, false, false>(p, s);
    return qlo ? launch_step<FMT, DP, NT, false, true, false>(p, s) : launch_step<FMT, DP, NT, false, false, false>(p, s);
}

template <int FMT>
int launch_step(const AttnParams& p, int nt, cudaStream_t s) {
    if (p.c.D > 128) return launch_step<FMT, 256, 1>(p, s);
    if (p.c.D > 64) return nt == 2 ? launch_step<FMT, 128, 2>(p, s) : launch_step<FMT, 128, 1>(p, s);
    return nt == 2 ? launch_step<FMT, 64, 2>(p, s) : launch_step<FMT, 64, 1>(p, s);
}

}  // namespace
}  // namespace q8
}  // namespace akv
