// C-ABI entry points of the rotary positions (declared in
// include/akv_rotary.h): argument validation, launch shapes, dispatch.
#include <cuda_runtime.h>

#include "akv_q8_step_launch.h"
#include "akv_rotary.cuh"

using namespace akv;

namespace {

template <typename T, int N>
void launch_rotate(const RotateParams& p, bool interleaved, unsigned blocks, cudaStream_t s) {
    if constexpr (N < 8) {  // interleaved, four pairs are 16 bytes
        if (interleaved) {
            rotate_kernel<T, N, true><<<blocks, kRotateThreads, 0, s>>>(p);
            return;
        }
    }
    rotate_kernel<T, N, false><<<blocks, kRotateThreads, 0, s>>>(p);
}

}  // namespace

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
    // The widest pieces that sizes and addresses allow: 8 pairs (16 bytes of
    // either half), 4 pairs, else one.
    const auto aligned = [&](int64_t bytes) {
        bool a = reinterpret_cast<uintptr_t>(p.x) % bytes == 0 && reinterpret_cast<uintptr_t>(p.out) % bytes == 0;
        for (const int64_t st : {p.xB, p.xT, p.xH, p.oB, p.oT, p.oH}) a = a && st * elem % bytes == 0;
        return a;
    };
    int N = 1;
    if (elem == 2 && !d->rotary.interleaved && p.r.R % 16 == 0 && p.D % 16 == 0 && aligned(16)) N = 8;
    else if (p.r.R % 8 == 0 && p.D % 8 == 0 && aligned(4 * elem)) N = 4;
    const int64_t tokens = static_cast<int64_t>(p.B) * p.n, units = (p.D + 2 * N - 1) / (2 * N);
    // Eight heads a thread where that leaves some waves of threads, fewer else.
    const int64_t few = static_cast<int64_t>(148) * 2048;
    int64_t splits = (p.H + 7) / 8;
    const int64_t want = (few + tokens * units - 1) / (tokens * units);
    if (splits < want) splits = want < p.H ? want : p.H;
    if (tokens * units * splits > 0x7FFFFF00) splits = 1;
    if (tokens * units * splits > 0x7FFFFF00) return AKV_ERR_UNSUPPORTED;
    p.splits = static_cast<int>(splits);
    const unsigned blocks = static_cast<unsigned>((tokens * units * splits + kRotateThreads - 1) / kRotateThreads);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool inter = d->rotary.interleaved != 0;
    if (d->dtype == AKV_Q_F32) {
        if (N == 4) launch_rotate<float, 4>(p, inter, blocks, s);
        else launch_rotate<float, 1>(p, inter, blocks, s);
    } else if (d->dtype == AKV_Q_BF16) {
        if (N == 8) launch_rotate<__nv_bfloat16, 8>(p, false, blocks, s);
        else if (N == 4) launch_rotate<__nv_bfloat16, 4>(p, inter, blocks, s);
        else launch_rotate<__nv_bfloat16, 1>(p, inter, blocks, s);
    } else {
        if (N == 8) launch_rotate<__half, 8>(p, false, blocks, s);
        else if (N == 4) launch_rotate<__half, 4>(p, inter, blocks, s);
        else launch_rotate<__half, 1>(p, inter, blocks, s);
    }
    return q8::launched();
}

}  // extern "C"
