// Template dispatch of the 4-bit cache's step kernel, included by akv_q4_step_*.cu.
#pragma once
#include "akv_q4_step.cuh"

namespace akv {
namespace q4 {
namespace {

template <int DP, int NT, bool PLO, bool QLO, bool TWIN, bool DENSE>
int launch(const Q4Params& p, cudaStream_t s) {
    if constexpr (NT == 1) {
        if (p.a.share_ctas < 0) {
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = static_cast<unsigned>(-p.a.share_ctas);
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(static_cast<unsigned>(p.c.B) * p.c.H * static_cast<unsigned>(-p.a.share_ctas));
            cfg.blockDim = dim3(kStepThreads);
            cfg.stream = s;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            return cudaLaunchKernelEx(&cfg, step_kernel<DP, 1, PLO, QLO, TWIN, true, DENSE, PLO>, p) == cudaSuccess
                       ? AKV_OK : (cudaGetLastError(), AKV_ERR_CUDA);
        }
    }
    if constexpr (!PLO) {
        if (p.a.long_sums) {
            step_kernel<DP, NT, PLO, QLO, TWIN, false, DENSE, true><<<p.a.share_ctas, kStepThreads, 0, s>>>(p);
            return q8::launched();
        }
    }
    step_kernel<DP, NT, PLO, QLO, TWIN, false, DENSE, PLO><<<p.a.share_ctas, kStepThreads, 0, s>>>(p);
    return q8::launched();
}

template <int DP, int NT, bool DENSE>
int launch(const Q4Params& p, cudaStream_t s) {
    const bool plo = p.a.out_dtype == AKV_Q_F32, qlo = p.a.q_dtype == AKV_Q_F32;
    if constexpr (NT == 1) {
        if (plo && p.a.R <= 4) return qlo ? launch<DP, 1, true, true, true, DENSE>(p, s) : launch<DP, 1, true, false, true, DENSE>(p, s);
    }
    if (plo) return qlo ? launch<DP, NT, true, true, false, DENSE>(p, s) : launch<DP, NT, true, false, false, DENSE>(p, s);
    return qlo ? launch<DP, NT, false, true, false, DENSE>(p, s) : launch<DP, NT, false, false, false, DENSE>(p, s);
}

template <bool DENSE>
int launch(const Q4Params& p, int nt, cudaStream_t s) {
    if (p.c.D > 128) return launch<256, 1, DENSE>(p, s);
    if (p.c.D > 64) return nt == 2 ? launch<128, 2, DENSE>(p, s) : launch<128, 1, DENSE>(p, s);
    return nt == 2 ? launch<64, 2, DENSE>(p, s) : launch<64, 1, DENSE>(p, s);
}

}  // namespace
}  // namespace q4
}  // namespace akv
