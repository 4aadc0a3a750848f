// C-ABI entry points of the rotary positions (declared in
// include/akv_rotary.h): argument validation, launch shapes, dispatch.
#include <cuda_runtime.h>

#include "akv_q8_step_launch.h"
#include "akv_rotary.cuh"

namespace akv {
namespace {

template <typename T, int N>
void launch(const RotateParams& p, bool interleaved, unsigned blocks, cudaStream_t s) {
    if constexpr (N < 8) {  // interleaved, four pairs are 16 bytes
        if (interleaved) {
            rotate_kernel<T, N, true><<<blocks, kRotateThreads, 0, s>>>(p);
            return;
        }
    }
    rotate_kernel<T, N, false><<<blocks, kRotateThreads, 0, s>>>(p);
}

}  // namespace

int launch_rotate(RotateParams p, int dtype, bool interleaved, cudaStream_t s) {
    const int N = rotate_width(p, interleaved, dtype == AKV_Q_F32 ? 4 : 2);
    p.splits = rotate_splits(p, N);
    if (p.splits == 0) return AKV_ERR_UNSUPPORTED;
    const int64_t threads = static_cast<int64_t>(p.B) * p.n * p.splits * ((p.D + 2 * N - 1) / (2 * N));
    const unsigned blocks = static_cast<unsigned>((threads + kRotateThreads - 1) / kRotateThreads);
    if (dtype == AKV_Q_F32) {
        if (N == 4) launch<float, 4>(p, interleaved, blocks, s);
        else launch<float, 1>(p, interleaved, blocks, s);
    } else if (dtype == AKV_Q_BF16) {
        if (N == 8) launch<__nv_bfloat16, 8>(p, false, blocks, s);
        else if (N == 4) launch<__nv_bfloat16, 4>(p, interleaved, blocks, s);
        else launch<__nv_bfloat16, 1>(p, interleaved, blocks, s);
    } else {
        if (N == 8) launch<__half, 8>(p, false, blocks, s);
        else if (N == 4) launch<__half, 4>(p, interleaved, blocks, s);
        else launch<__half, 1>(p, interleaved, blocks, s);
    }
    return q8::launched();
}

}  // namespace akv

using namespace akv;

extern "C" {

size_t akv_rotary_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(AkvRotary);
        case 1: return sizeof(AkvRotateDesc);
        default: return 0;
    }
}

int akv_rotate(const AkvRotateDesc* d, void* stream) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (d->batch < 0 || d->tokens < 0 || d->heads <= 0 || d->head_dim <= 0 || d->dtype < AKV_Q_F32 || d->dtype > AKV_Q_F16)
        return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_rotary(d->rotary, d->head_dim)) return st;
    if (d->head_dim > 256) return AKV_ERR_UNSUPPORTED;
    if (d->batch == 0 || d->tokens == 0) return AKV_OK;
    const int64_t elem = d->dtype == AKV_Q_F32 ? 4 : 2;
    if (!d->x_dev || !d->out_dev || !d->positions_dev || reinterpret_cast<uintptr_t>(d->x_dev) % elem ||
        reinterpret_cast<uintptr_t>(d->out_dev) % elem || reinterpret_cast<uintptr_t>(d->positions_dev) % 4 ||
        reinterpret_cast<uintptr_t>(d->status_dev) % 4)
        return AKV_ERR_INVALID_ARGUMENT;
    RotateParams p;
    p.r = to_dev(d->rotary);
    p.B = d->batch; p.n = d->tokens; p.H = d->heads; p.D = d->head_dim;
    p.inverse = d->inverse != 0;
    p.x = d->x_dev; p.out = d->out_dev;
    p.xB = d->x_stride[0]; p.xT = d->x_stride[1]; p.xH = d->x_stride[2];
    p.oB = d->out_stride[0]; p.oT = d->out_stride[1]; p.oH = d->out_stride[2];
    p.places = d->positions_dev; p.status = d->status_dev;
    p.start = p.counts = nullptr;
    return launch_rotate(p, d->dtype, d->rotary.interleaved != 0, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
