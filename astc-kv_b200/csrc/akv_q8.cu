// C-ABI entry points of the 8-bit KV cache (declared in include/akv_q8.h):
// argument validation, launch shapes, template dispatch.
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <initializer_list>

#include "../../include/akv_q8.h"
#include "akv_q8_attend.cuh"
#include "akv_q8_chunk.cuh"
#include "akv_q8_evict.cuh"
#include "akv_q8_step_launch.h"
#include "akv_q8_store.cuh"
#include "akv_q8_weights.cuh"

namespace akv {
namespace q8 {
namespace {

constexpr int kMaxGridYZ = 65535;


bool valid_dtype(int t) { return t >= AKV_Q_F32 && t <= AKV_Q_F16; }

// Words that kernels read or write one at a time, or NULL.
bool words(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % 4) return false;
    return true;
}

// A cache for no sequences needs no memory.
bool valid_side(const AkvQ8Side& s, int batch) {
    return (batch == 0 || (s.codes && s.scales)) && reinterpret_cast<uintptr_t>(s.codes) % 16 == 0 && reinterpret_cast<uintptr_t>(s.scales) % 4 == 0 &&
           s.stride_batch % 16 == 0 && s.stride_head % 16 == 0 && s.stride_page % 16 == 0 && s.stride_token % 16 == 0;
}

int check_cache(const AkvQ8Cache& c) {
    if (c.format != AKV_Q8_INT8 && c.format != AKV_Q8_E4M3) return AKV_ERR_INVALID_ARGUMENT;
    if (c.batch < 0 || c.kv_heads <= 0 || c.head_dim <= 0 || c.max_tokens <= 0 || c.page_tokens <= 0) return AKV_ERR_INVALID_ARGUMENT;
    if (!valid_side(c.k, c.batch) || !valid_side(c.v, c.batch) || !words({c.block_table_dev, c.status_dev})) return AKV_ERR_INVALID_ARGUMENT;
    if (c.block_tokens <= 0 || c.page_tokens % c.block_tokens) return AKV_ERR_INVALID_ARGUMENT;
    if (c.block_table_dev &&
        (c.pages_per_seq <= 0 || c.num_pages <= 0 || static_cast<int64_t>(c.pages_per_seq) * c.page_tokens < c.max_tokens))
        return AKV_ERR_INVALID_ARGUMENT;
    if (c.block_tokens != 16 && c.block_tokens != 32 && c.block_tokens != 64 && c.block_tokens != 128) return AKV_ERR_UNSUPPORTED;
    if (c.head_dim % 16 || c.head_dim > 256 || c.kv_heads > kMaxGridYZ || c.batch > kMaxGridYZ / 2 ||
        c.max_tokens > 1 << 30)
        return AKV_ERR_UNSUPPORTED;
    return AKV_OK;
}

// Launches a kernel that calls wait_for_previous_kernel() so that it may be
// brought onto the SMs while the kernel before it ends.
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t s, A... args) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess ? AKV_OK : (cudaGetLastError(), AKV_ERR_CUDA);
}

// Calls fn with a value of the element type of an AKV_Q_* code.
template <typename F>
void with_type(int dtype, F fn) {
    if (dtype == AKV_Q_F32) fn(float{});
    else if (dtype == AKV_Q_BF16) fn(__nv_bfloat16{});
    else fn(__half{});
}

int check_attention(const AkvQ8AttnDesc* d) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->cache)) return st;
    if (d->q_heads <= 0 || d->q_heads % d->cache.kv_heads || d->q_tokens < 0 || !valid_dtype(d->q_dtype) || !valid_dtype(d->out_dtype))
        return AKV_ERR_INVALID_ARGUMENT;
    if (d->split_tokens < 0 || d->split_tokens % 16 || !(d->scale >= 0.f) || std::isinf(d->scale)) return AKV_ERR_INVALID_ARGUMENT;
    if (d->weights_dev && d->weights_stride < d->cache.max_tokens) return AKV_ERR_INVALID_ARGUMENT;
    if (!words({d->seq_lens_dev, d->q_lens_dev, d->lse_dev, d->weights_dev})) return AKV_ERR_INVALID_ARGUMENT;
    const int64_t rows = static_cast<int64_t>(d->q_heads) * d->q_tokens;
    if (rows > 1 << 24 || rows * d->cache.batch > 1 << 30) return AKV_ERR_UNSUPPORTED;
    return AKV_OK;
}

// SMs of the current device, asked once per device.
int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
    if (dev >= 0 && dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) cudaGetLastError();
    if (n <= 0) return 148;
    if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

struct AttnPlan {
    int rows;         // per kv head
    bool chunk;       // the tcgen05 kernel, else the step kernel
    int cluster;      // CTAs of the step kernel's clusters, 0 without
    int nt;           // groups of eight rows per CTA
    int split, nsplits;          // chunk kernel
    int share_ctas, share_min;   // step kernel
    bool long_sums;              // see kStepLong
    bool keep_scores; // the step kernel stores its scores for the token weights
    size_t part_ml, part_o, scores, lse, q_rows, q_factors, bytes;  // offsets into the workspace, and its size
};

// Rows from which the tcgen05 kernel, whose CTA does 128 or 256 rows for the
// price of one, is ahead of the step kernel, which does 16 at a time (8 above
// head_dim 128). Measured, 8 kv heads, step kernel against tcgen05, B8 x 8192
// tokens: D 128 int8 20 rows 78 us against 81, 32 rows 81 against 82, 36 rows
// 109 against 82; D 64 32 rows 50 against 59, 36 rows 67 against 60; D 256 int8 16 rows 106 against
// 119, 20 rows 143 against 120, e4m3 101 against 114 and 134 against 115.
// (B1 x 32768, D 128, 32 rows 47 against 43; B8 x 700, D 64, 20 rows 20
// against 17: short of 33 rows neither is far ahead up to D 128.)
int chunk_min_rows(int head_dim) { return head_dim <= 128 ? 33 : 17; }

// Tokens that a tile of the tcgen05 kernel adds up at most, also where a caller
// asks for longer splits. The tensor cores truncate as they add: a sum over n tokens comes out
// 6e-9 n too small (measured: 3e-5 at 8192, 8e-4 at 131072, 6.7e-3 at a million tokens), which fp16
// outputs, 2.4e-4 off by their rounding on the average, would show, and bf16
// ones, which are eight times coarser, later. A second
// partial costs about 2.5 of this split's 128 steps.
constexpr int64_t kChunkHalfTokens = 16384, kChunkBf16Tokens = 131072;

// Tokens for each CTA of a cluster up to which a cluster for each kv head of
// each sequence beats even shares of all CTAs and a second launch (32/8 heads:
// B1 x 4096 in clusters of eight 16.0 us against 18.8; B64 x 300, a CTA each,
// 22 against 30, the same ragged to 500 tokens 19 against 27).
constexpr int kClusterTokens = 512;

// Scores are stored for the token weights, rather than computed again, where one
// CTA of the step kernel has all rows. Storing costs 8 bytes per row
// and token, a second pass over K head_dim bytes per token and the products;
// stored against computed, B8 x 8192 tokens, 8 kv heads, int8: D 64 1 row 28 us
// against 59, 16 rows 52 against 71; D 128 41 against 93 and 66 against 109;
// D 256 8 rows 72 against 177. Stored scores take 4 bytes of workspace per row,
// kv head and token of max_tokens.
bool keeps_scores(const AttnPlan& a) { return !a.chunk && a.rows <= 8 * a.nt; }

AttnPlan plan_attention(const AkvQ8AttnDesc* d) {
    AttnPlan a = {};
    const AkvQ8Cache& c = d->cache;
    const int64_t bh = static_cast<int64_t>(c.batch) * c.kv_heads;
    a.rows = d->q_tokens * (d->q_heads / c.kv_heads);
    a.nt = c.head_dim <= 128 && a.rows > 8 ? 2 : 1;
    a.chunk = a.rows >= chunk_min_rows(c.head_dim) && d->q_dtype != AKV_Q_F32 && d->out_dtype != AKV_Q_F32;
    a.keep_scores = d->weights_dev && keeps_scores(a);
    a.split = d->split_tokens;
    const bool shared = a.chunk && a.rows <= 128 && c.head_dim <= 128;  // its two tiles share the rows and take every other step
    const int group = a.chunk ? (c.head_dim <= 128 ? 256 : 128) : 8 * a.nt;  // rows of a CTA
    // (Two tiles that take every other step share a split.)
    const int64_t longest = (d->out_dtype == AKV_Q_F16 ? kChunkHalfTokens : kChunkBf16Tokens) * (shared ? 2 : 1);
    if (a.split == 0 && a.chunk) {
        // One CTA per SM. In steps of 128 tokens a CTA costs its share of the
        // tokens, about three to start and, when split, 2.5 (D 128) for a
        // partial written and read; the number of splits, up to eight or one
        // wave, is that of the least cost over the waves. Where lengths may be
        // ragged more splits are taken for up to 15 %: short sequences then
        // leave SMs to long ones. 4 x 128 query tokens, 32/8 heads, D 128, up
        // to 8192 tokens, four splits against two: 241 to 8192 tokens 67 us
        // against 100, all 8192 119 against 103; 4 x 509, 9/3 heads, D 64: 58
        // against 89, and 100 against 90. Not where units fill the SMs, which
        // then even the lengths out by themselves: 4 x 512 query tokens, four
        // splits against one, ragged 234 against 159, equal 425 against 313.
        const int64_t units = bh * ((a.rows + group - 1) / group), sms = sm_count();
        const int64_t steps = (static_cast<int64_t>(c.max_tokens) + kChunkTokens - 1) / kChunkTokens;
        const int64_t most = units > 0 && sms / units > 8 ? sms / units : 8;
        const auto cost = [&](int64_t n) {
            const double each = static_cast<double>((steps + n - 1) / n) + 3.0 + (n > 1 ? 2.5 * c.head_dim / 128 : 0.0);
            return static_cast<double>((units * n + sms - 1) / sms) * each;
        };
        double least = cost(1);
        for (int64_t n = 2; n <= most && n <= steps; ++n) least = cost(n) < least ? cost(n) : least;
        int64_t best = 1;
        const double limit = d->seq_lens_dev && c.batch > 1 && units < sms ? 1.15 * least : least;
        for (int64_t n = 2; n <= most && n <= steps; ++n)
            if (cost(n) <= limit) best = n;
        if (cost(1) <= least) best = best > 1 && limit > least ? best : 1;
        const int64_t n = (steps * kChunkTokens + longest - 1) / longest;
        best = best > n ? best : n;
        a.split = static_cast<int>((steps + best - 1) / best * kChunkTokens);
    }
    size_t parts;  // rows of partials
    if (a.chunk) {
        if (a.split > longest) a.split = static_cast<int>(longest);
        // Whole steps: a step's tokens past the split's end would count as seen.
        a.split = static_cast<int>((static_cast<int64_t>(a.split < c.max_tokens ? a.split : c.max_tokens) + kChunkTokens - 1) / kChunkTokens * kChunkTokens);
        a.nsplits = static_cast<int>((static_cast<int64_t>(c.max_tokens) + a.split - 1) / a.split);
        const int64_t limit = 0x7FFFFFFF / ((a.rows + group - 1) / group + 1);
        while (a.nsplits > limit) {  // the grid holds splits x row groups
            a.split *= 2;
            a.nsplits = static_cast<int>((static_cast<int64_t>(c.max_tokens) + a.split - 1) / a.split);
        }
        if (shared) a.nsplits *= 2;
        parts = a.nsplits > 1 ? static_cast<size_t>(bh) * a.nsplits * a.rows : 0;
    } else {
        // One wave of CTAs (see the step kernel), two pieces each; no more
        // CTAs than there can be chunks.
        const int64_t chunks = bh * ((a.rows + group - 1) / group) * ((c.max_tokens + kShareTokens - 1) / kShareTokens);
        const int64_t slots = static_cast<int64_t>(sm_count()) * (c.head_dim > 128 || a.nt == 2 ? 2 : 4);
        a.share_min = a.split > kShareTokens ? a.split / kShareTokens : 1;
        const int64_t ctas = chunks / a.share_min < slots ? chunks / a.share_min : slots;
        a.share_ctas = static_cast<int>(ctas > 0 ? ctas : 1);
        a.nsplits = 0;
        a.long_sums = step_sums_long(chunks, a.share_ctas, a.share_min, c.max_tokens, d->out_dtype);
        parts = 2 * static_cast<size_t>(a.share_ctas) * group;
        // The largest cluster with which all units fit the GPU at once.
        int size = kStepCluster;
        while (size > 1 && bh * size > slots) size /= 2;
        a.cluster = a.split == 0 && a.rows <= 8 && c.max_tokens <= kClusterTokens * size ? size : 0;
    }
    const auto up = [](size_t x) { return (x + 15) / 16 * 16; };
    a.part_ml = 0;
    a.part_o = up(parts * sizeof(float2));
    a.scores = a.part_o + up(parts * c.head_dim * sizeof(float));
    a.lse = a.scores + (a.keep_scores ? up(static_cast<size_t>(bh) * c.max_tokens * a.rows * sizeof(float)) : 0);
    a.q_rows = a.lse + (d->weights_dev ? up(static_cast<size_t>(c.batch) * d->q_tokens * d->q_heads * sizeof(float)) : 0);
    a.q_factors = a.q_rows;
    a.bytes = a.q_rows + 16;
    if (d->weights_dev && !a.keep_scores) {
        const size_t groups = static_cast<size_t>(bh) * ((a.rows + 7) / 8), dim = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
        a.q_factors = a.q_rows + groups * 8 * dim * 2 * (d->q_dtype == AKV_Q_F32 ? 2 : 1);
        a.bytes = a.q_factors + groups * 8 * sizeof(float) + 16;
    }
    return a;
}

template <int FMT, int DP, bool SHARED>
int launch_chunk(const AttnParams& p, cudaStream_t s) {
    const auto kern = chunk_kernel<FMT, DP, SHARED>;
    constexpr int bytes = sizeof(ChunkSmem<DP>) + 1024;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return AKV_ERR_CUDA;
    }
    const int parts = SHARED ? p.nsplits / 2 : p.nsplits;
    constexpr int rows = 128 * kChunkTiles<DP>;
    const dim3 grid(parts * ((p.R + rows - 1) / rows), p.c.H, p.c.B);
    kern<<<grid, kChunkThreads<DP>, bytes, s>>>(p);
    return launched();
}

template <int FMT>
int launch_chunk(const AttnParams& p, cudaStream_t s) {
    if (p.c.D > 128) return launch_chunk<FMT, 256, false>(p, s);
    if (p.R <= 128) return p.c.D > 64 ? launch_chunk<FMT, 128, true>(p, s) : launch_chunk<FMT, 64, true>(p, s);
    return p.c.D > 64 ? launch_chunk<FMT, 128, false>(p, s) : launch_chunk<FMT, 64, false>(p, s);
}

template <int FMT, int DP>
int launch_weights(const AttnParams& p, cudaStream_t s) {
    const dim3 grid((p.c.T + kWeightTile - 1) / kWeightTile, p.c.H, p.c.B);
    if (p.q_dtype == AKV_Q_F32) return launch_after(weights_kernel<FMT, DP, true>, grid, kWeightThreads, s, p);
    return launch_after(weights_kernel<FMT, DP, false>, grid, kWeightThreads, s, p);
}

template <int FMT>
int launch_weights(const AttnParams& p, cudaStream_t s) {
    if (p.c.D > 128) return launch_weights<FMT, 256>(p, s);
    if (p.c.D > 64) return launch_weights<FMT, 128>(p, s);
    return launch_weights<FMT, 64>(p, s);
}

}  // namespace
}  // namespace q8
}  // namespace akv

using namespace akv;
using namespace akv::q8;

extern "C" {

size_t akv_q8_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(AkvQ8Cache);
        case 1: return sizeof(AkvQ8StoreDesc);
        case 2: return sizeof(AkvQ8RestoreDesc);
        case 3: return sizeof(AkvQ8AttnDesc);
        case 4: return sizeof(AkvQ8EvictDesc);
        default: return 0;
    }
}

int akv_q8_store(const AkvQ8StoreDesc* d, void* stream) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->cache)) return st;
    if (d->tokens < 0 || !valid_dtype(d->dtype)) return AKV_ERR_INVALID_ARGUMENT;
    if (d->cache.batch == 0 || d->tokens == 0) return AKV_OK;
    const uintptr_t elem = d->dtype == AKV_Q_F32 ? 4 : 2;
    if (!d->k_dev || !d->v_dev || !d->start_dev || reinterpret_cast<uintptr_t>(d->k_dev) % elem ||
        reinterpret_cast<uintptr_t>(d->v_dev) % elem || !words({d->start_dev, d->counts_dev}))
        return AKV_ERR_INVALID_ARGUMENT;
    StoreParams p;
    p.c = to_dev(d->cache);
    p.x[0] = d->k_dev; p.x[1] = d->v_dev;
    p.xB[0] = d->k_stride[0]; p.xT[0] = d->k_stride[1]; p.xH[0] = d->k_stride[2];
    p.xB[1] = d->v_stride[0]; p.xT[1] = d->v_stride[1]; p.xH[1] = d->v_stride[2];
    p.start = d->start_dev; p.counts = d->counts_dev; p.n = d->tokens;
    for (int i = 0; i < 2; ++i) {
        p.vec[i] = reinterpret_cast<uintptr_t>(p.x[i]) % 16 == 0;
        for (const int64_t st : {p.xB[i], p.xT[i], p.xH[i]}) p.vec[i] = p.vec[i] && st * static_cast<int64_t>(elem) % 16 == 0;
    }
    const int blocks = static_cast<int>((static_cast<int64_t>(d->tokens) + 2 * p.c.blk - 2) / p.c.blk);
    const dim3 grid(blocks, p.c.H, 2 * p.c.B);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    // A block's new rows in pieces: a few threads for a few rows (one token,
    // B64, 8 heads, D 128: 2.7 us against 4.1 with 256 threads; B512 7.9
    // against 19.6), else 256 with two or eight pieces each.
    const int pieces = (d->tokens < p.c.blk ? d->tokens : p.c.blk) * (p.c.D / 16);
    const int threads = pieces <= 128 ? 64 : 256;
    with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        const bool few = pieces <= 2 * threads;
        if (p.c.fmt == AKV_Q8_INT8) {
            if (few) store_kernel<AKV_Q8_INT8, T, 2><<<grid, threads, 0, s>>>(p);
            else store_kernel<AKV_Q8_INT8, T, 8><<<grid, threads, 0, s>>>(p);
        } else {
            if (few) store_kernel<AKV_Q8_E4M3, T, 2><<<grid, threads, 0, s>>>(p);
            else store_kernel<AKV_Q8_E4M3, T, 8><<<grid, threads, 0, s>>>(p);
        }
    });
    return launched();
}

int akv_q8_restore(const AkvQ8RestoreDesc* d, void* stream) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->cache)) return st;
    if (d->tokens < 0 || !valid_dtype(d->dtype)) return AKV_ERR_INVALID_ARGUMENT;
    if (d->cache.batch == 0 || d->tokens == 0) return AKV_OK;
    if (!d->k_dev || !d->v_dev || reinterpret_cast<uintptr_t>(d->k_dev) % 16 || reinterpret_cast<uintptr_t>(d->v_dev) % 16 || !words({d->start_dev}))
        return AKV_ERR_INVALID_ARGUMENT;
    RestoreParams p;
    p.c = to_dev(d->cache);
    p.out[0] = d->k_dev; p.out[1] = d->v_dev;
    p.start = d->start_dev; p.n = d->tokens;
    const int64_t pieces = static_cast<int64_t>(p.n) * p.c.H * (p.c.D / 16);  // of a sequence's side
    if (pieces > 0x7FFFFFFF) return AKV_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>((pieces + 255) / 256), 2 * p.c.B);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int st = AKV_OK;
    with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        if (p.c.fmt == AKV_Q8_INT8) st = launch_after(restore_kernel<AKV_Q8_INT8, T>, grid, 256, s, p);
        else st = launch_after(restore_kernel<AKV_Q8_E4M3, T>, grid, 256, s, p);
    });
    return st;
}

size_t akv_q8_attention_workspace(const AkvQ8AttnDesc* d) { return check_attention(d) == AKV_OK ? plan_attention(d).bytes : 0; }

int akv_q8_attention(const AkvQ8AttnDesc* d, void* stream) {
    if (int st = check_attention(d)) return st;
    if (d->cache.batch == 0) return AKV_OK;
    if (d->q_tokens == 0) {
        // A sum over no queries.
        if (!d->weights_dev || d->accumulate) return AKV_OK;
        const AkvQ8Cache& c = d->cache;
        return cudaMemset2DAsync(d->weights_dev, d->weights_stride * sizeof(float), 0, c.max_tokens * sizeof(float),
                                 static_cast<size_t>(c.batch) * c.kv_heads, static_cast<cudaStream_t>(stream)) == cudaSuccess
                   ? AKV_OK : (cudaGetLastError(), AKV_ERR_CUDA);
    }
    const uintptr_t elem = d->q_dtype == AKV_Q_F32 ? 4 : 2;
    if (!d->q_dev || !d->out_dev || reinterpret_cast<uintptr_t>(d->q_dev) % elem || reinterpret_cast<uintptr_t>(d->out_dev) % 16)
        return AKV_ERR_INVALID_ARGUMENT;
    const AttnPlan plan = plan_attention(d);
    if (!d->workspace_dev || d->workspace_bytes < plan.bytes) return AKV_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(d->workspace_dev) % 16) return AKV_ERR_INVALID_ARGUMENT;
    char* ws = static_cast<char*>(d->workspace_dev);
    AttnParams p;
    p.c = to_dev(d->cache);
    p.Hq = d->q_heads; p.G = d->q_heads / d->cache.kv_heads; p.n = d->q_tokens; p.R = plan.rows;
    p.q_dtype = d->q_dtype; p.out_dtype = d->out_dtype; p.causal = d->causal; p.accumulate = d->accumulate;
    p.q_vec = reinterpret_cast<uintptr_t>(d->q_dev) % 16 == 0;
    for (int i = 0; i < 3; ++i) p.q_vec &= d->q_stride[i] * static_cast<int64_t>(elem) % 16 == 0;
    p.c2 = (d->scale > 0.f ? d->scale : 1.0f / std::sqrt(static_cast<float>(p.c.D))) * 1.4426950408889634f;
    p.q = d->q_dev; p.qB = d->q_stride[0]; p.qT = d->q_stride[1]; p.qH = d->q_stride[2];
    p.lens = d->seq_lens_dev; p.q_lens = d->q_lens_dev;
    p.split = plan.split; p.nsplits = plan.nsplits;
    p.share_ctas = plan.chunk ? 0 : plan.cluster ? -plan.cluster : plan.share_ctas; p.share_min = plan.share_min; p.row_group = 8 * plan.nt;
    p.long_sums = plan.long_sums;
    p.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
    p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
    p.scores = plan.keep_scores ? reinterpret_cast<float*>(ws + plan.scores) : nullptr;
    p.lse = d->weights_dev ? reinterpret_cast<float*>(ws + plan.lse) : nullptr;
    p.q_rows = reinterpret_cast<uint2*>(ws + plan.q_rows);
    p.q_factors = reinterpret_cast<float*>(ws + plan.q_factors);
    p.out = d->out_dev; p.lse_out = d->lse_dev;
    p.weights = d->weights_dev; p.wstride = d->weights_stride;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool int8 = p.c.fmt == AKV_Q8_INT8;
    if (int st = plan.chunk ? (int8 ? launch_chunk<AKV_Q8_INT8>(p, s) : launch_chunk<AKV_Q8_E4M3>(p, s))
                            : (int8 ? launch_step_int8(p, plan.nt, s) : launch_step_e4m3(p, plan.nt, s)))
        return st;
    // A step kernel of one CTA leaves nothing to combine.
    const bool combine = plan.chunk ? plan.nsplits > 1 : !plan.cluster && plan.share_ctas > 1;
    const int64_t rows = combine ? static_cast<int64_t>(p.c.B) * p.c.H * p.R : 0;
    // Tokens per CTA of the weights part: one wave of CTAs where there are
    // tokens enough, since each first works out the rows' log-sum-exps (B2,
    // 131071 tokens: 126 us the whole call, with four times the CTAs 133).
    int wtokens = kCombineThreads;
    while (wtokens < 8192 && static_cast<int64_t>(p.c.B) * p.c.H * p.c.T / wtokens > 4 * sm_count()) wtokens *= 2;
    const int wblocks = plan.keep_scores ? (p.c.T + wtokens - 1) / wtokens : 0;
    // Partials of a row: of all rows alike, or as the shares fall. A warp a
    // row where they are few (B64 x 300 tokens, 32/8 heads: 30 us the whole
    // call, with a CTA a row 42).
    const int64_t pieces = plan.chunk ? plan.nsplits : plan.share_ctas / (static_cast<int64_t>(p.c.B) * p.c.H) + 1;
    const bool by_warp = pieces <= 16 && rows >= 1024;
    constexpr int per = kCombineThreads / 32;
    const bool recompute = p.weights && !plan.keep_scores;
    const int64_t packs = recompute ? static_cast<int64_t>(p.c.B) * p.c.H * ((p.R + 7) / 8) : 0;
    const int64_t blocks = (by_warp ? (rows + per - 1) / per : rows) + (packs + per - 1) / per + static_cast<int64_t>(p.c.B) * p.c.H * wblocks;
    if (blocks) {
        if (int st = launch_after(combine_kernel, dim3(static_cast<unsigned>(blocks)), kCombineThreads, s, p, static_cast<int>(rows), by_warp,
                                  wblocks, wtokens, static_cast<int>(packs)))
            return st;
    }
    if (recompute) return int8 ? launch_weights<AKV_Q8_INT8>(p, s) : launch_weights<AKV_Q8_E4M3>(p, s);
    return AKV_OK;
}

int akv_q8_evict(const AkvQ8EvictDesc* d, void* stream) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->src)) return st;
    if (int st = check_cache(d->dst)) return st;
    const AkvQ8Cache &a = d->src, &c = d->dst;
    if (a.format != c.format || a.batch != c.batch || a.kv_heads != c.kv_heads || a.head_dim != c.head_dim) return AKV_ERR_INVALID_ARGUMENT;
    if (d->keep <= 0 || d->keep > c.max_tokens || d->sinks < 0 || d->recent < 0 ||
        static_cast<int64_t>(d->sinks) + d->recent > d->keep)
        return AKV_ERR_INVALID_ARGUMENT;
    if (d->out_weights_tokens && (d->out_weights_tokens < d->keep || d->out_weights_tokens > d->out_weights_stride)) return AKV_ERR_INVALID_ARGUMENT;
    if (d->weights_stride < a.max_tokens || d->out_weights_stride < d->keep) return AKV_ERR_INVALID_ARGUMENT;
    // Two tables may give out pages of one pool.
    const auto same = [](const void* x, const void* y) { return x && x == y; };
    if (!(a.block_table_dev && c.block_table_dev && a.block_table_dev != c.block_table_dev) &&
        (same(a.k.codes, c.k.codes) || same(a.v.codes, c.v.codes) || same(a.k.scales, c.k.scales) || same(a.v.scales, c.v.scales)))
        return AKV_ERR_INVALID_ARGUMENT;
    if (a.batch == 0) return AKV_OK;
    if (!d->weights_dev || !d->kept_dev || !d->out_lens_dev || !d->out_weights_dev ||
        !words({d->weights_dev, d->kept_dev, d->out_lens_dev, d->out_weights_dev, d->seq_lens_dev}))
        return AKV_ERR_INVALID_ARGUMENT;
    EvictParams p;
    p.src = to_dev(a); p.dst = to_dev(c);
    p.weights = d->weights_dev; p.wstride = d->weights_stride; p.lens = d->seq_lens_dev;
    p.keep = d->keep; p.sinks = d->sinks; p.recent = d->recent;
    p.columns = d->out_weights_tokens ? d->out_weights_tokens : d->keep;
    p.kept = d->kept_dev; p.out_lens = d->out_lens_dev; p.out_weights = d->out_weights_dev; p.ostride = d->out_weights_stride;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.max_tokens <= 8 * kSelectThreads) select_kernel<8><<<dim3(a.kv_heads, a.batch), kSelectThreads, 0, s>>>(p);
    else select_kernel<32><<<dim3(a.kv_heads, a.batch), kSelectThreads, 0, s>>>(p);
    if (int st = launched()) return st;
    const dim3 grid((p.keep + p.dst.blk - 1) / p.dst.blk, a.kv_heads, a.batch);
    const bool few = c.block_tokens * (c.head_dim / 16) <= 512;  // pieces of a block
    if (a.format == AKV_Q8_INT8)
        return few ? launch_after(pack_kernel<AKV_Q8_INT8, 2>, grid, 256, s, p) : launch_after(pack_kernel<AKV_Q8_INT8, 8>, grid, 256, s, p);
    return few ? launch_after(pack_kernel<AKV_Q8_E4M3, 2>, grid, 256, s, p) : launch_after(pack_kernel<AKV_Q8_E4M3, 8>, grid, 256, s, p);
}

}  // extern "C"
