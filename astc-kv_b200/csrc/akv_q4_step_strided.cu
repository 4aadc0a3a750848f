// The 4-bit cache's step kernel for rows of codes that are any distance apart, and head_dims that are rounded up.
#include "akv_q4_step_launch.cuh"

int akv::q4::launch_step_strided(const Q4Params& p, int nt, cudaStream_t s) { return launch<false>(p, nt, s); }
