// The 4-bit cache's step kernel for rows of codes that follow one another.
#include "akv_q4_step_launch.cuh"

int akv::q4::launch_step_dense(const Q4Params& p, int nt, cudaStream_t s) { return launch<true>(p, nt, s); }
