// Template dispatch of the 4-bit cache's step kernel.
#include "akv_q4_step.cuh"

namespace akv {
namespace q4 {
namespace {

template <int DP, int NT, bool PLO, bool QLO, bool TWIN>
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
            return cudaLaunchKernelEx(&cfg, step_kernel<DP, 1, PLO, QLO, TWIN, true>, p) == cudaSuccess
                       ? AKV_OK : (cudaGetLastError(), AKV_ERR_CUDA);
        }
    }
    step_kernel<DP, NT, PLO, QLO, TWIN, false><<<p.a.share_ctas, kStepThreads, 0, s>>>(p);
    return q8::launched();
}

template <int DP, int NT>
int launch(const Q4Params& p, cudaStream_t s) {
    const bool plo = p.a.out_dtype == AKV_Q_F32, qlo = p.a.q_dtype == AKV_Q_F32;
    if constexpr (NT == 1) {
        if (plo && p.a.R <= 4) return qlo ? launch<DP, 1, true, true, true>(p, s) : launch<DP, 1, true, false, true>(p, s);
    }
    if (plo) return qlo ? launch<DP, NT, true, true, false>(p, s) : launch<DP, NT, true, false, false>(p, s);
    return qlo ? launch<DP, NT, false, true, false>(p, s) : launch<DP, NT, false, false, false>(p, s);
}

}  // namespace

int launch_step(const Q4Params& p, int nt, cudaStream_t s) {
    if (p.c.D > 128) return launch<256, 1>(p, s);
    if (p.c.D > 64) return nt == 2 ? launch<128, 2>(p, s) : launch<128, 1>(p, s);
    return nt == 2 ? launch<64, 2>(p, s) : launch<64, 1>(p, s);
}

}  // namespace q4
}  // namespace akv
