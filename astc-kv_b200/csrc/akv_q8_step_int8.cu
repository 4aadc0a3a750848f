// The step kernel for int8 codes.
#include "akv_q8_step_launch.cuh"

int akv::q8::launch_step_int8(const AttnParams& p, int nt, cudaStream_t s) { return launch_step<AKV_Q8_INT8>(p, nt, s); }
