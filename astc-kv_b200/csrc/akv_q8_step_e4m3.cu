// The step kernel for e4m3 codes.
#include "akv_q8_step_launch.cuh"

int akv::q8::launch_step_e4m3(const AttnParams& p, int nt, cudaStream_t s) { return launch_step<AKV_Q8_E4M3>(p, nt, s); }
