// C-ABI entry points of the 4-bit KV cache (declared in include/akv_q4.h):
// argument validation, launch shapes, template dispatch.
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <initializer_list>

#include "akv_q4_append.cuh"
#include "akv_q4_attend.cuh"
#include "akv_q4_chunk.cuh"

namespace akv {
namespace q4 {
namespace {

constexpr int kMaxGridYZ = 65535;

bool valid_dtype(int t) { return t >= AKV_Q_F32 && t <= AKV_Q_F16; }
int64_t size_of(int dtype) { return dtype == AKV_Q_F32 ? 4 : 2; }
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Words that kernels read or write one at a time, or NULL.
bool words(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (!aligned(p, 4)) return false;
    return true;
}

// A cache for no sequences needs no memory.
bool valid_side(const AkvQ4Side& s, int batch) {
    for (const int64_t st : {s.stride_batch, s.stride_head, s.stride_page, s.stride_token})
        if (st % 16) return false;
    for (const int64_t st : {s.scale_stride_batch, s.scale_stride_head, s.scale_stride_page, s.scale_stride_group})
        if (st % 4) return false;
    return (batch == 0 || (s.codes && s.scales)) && aligned(s.codes, 16) && aligned(s.scales, 8);
}

int check_cache(const AkvQ4Cache& c) {
    if (c.batch < 0 || c.kv_heads <= 0 || c.head_dim <= 0 || c.max_tokens <= 0 || c.page_tokens <= 0) return AKV_ERR_INVALID_ARGUMENT;
    if (!valid_side(c.k, c.batch) || !valid_side(c.v, c.batch) || !words({c.block_table_dev, c.status_dev})) return AKV_ERR_INVALID_ARGUMENT;
    if (c.page_tokens % AKV_Q4_TOKENS) return AKV_ERR_INVALID_ARGUMENT;
    if (c.block_table_dev &&
        (c.pages_per_seq <= 0 || c.num_pages <= 0 || static_cast<int64_t>(c.pages_per_seq) * c.page_tokens < c.max_tokens))
        return AKV_ERR_INVALID_ARGUMENT;
    if (c.head_dim % AKV_Q4_GROUP || c.head_dim > 256 || c.kv_heads > kMaxGridYZ || c.batch > kMaxGridYZ / 2 || c.max_tokens > 1 << 30)
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

int check_attention(const AkvQ4AttnDesc* d) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->cache)) return st;
    if (d->q_heads <= 0 || d->q_heads % d->cache.kv_heads || d->q_tokens < 0 || !valid_dtype(d->q_dtype) || !valid_dtype(d->out_dtype))
        return AKV_ERR_INVALID_ARGUMENT;
    if (d->split_tokens < 0 || d->split_tokens % 16 || d->wait_tries < 0 || !(d->scale >= 0.f) || std::isinf(d->scale)) return AKV_ERR_INVALID_ARGUMENT;
    if (!words({d->seq_lens_dev, d->q_lens_dev, d->lse_dev})) return AKV_ERR_INVALID_ARGUMENT;
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
    bool long_sums;              // see q8::kStepLong
    size_t part_ml, part_o, bytes;  // offsets into the workspace, and its size
};

// Rows from which the tcgen05 kernel is taken, whose CTA does 128 or 256 rows
// for the price of one, rather than the step kernel, which does 16 at a time
// (8 above head_dim 128) and starts sooner. Measured, step and chunk kernel in us:
//   head_dim 128, 8 heads, 32768 tokens      20 rows 37, 34   32 rows 38, 35   40 rows 47, 35
//   head_dim 128, 8 x 8 heads, 8192 tokens   20 rows 57, 66   32 rows 60, 68   40 rows 81, 69
//   head_dim 128, 2 x 8 heads, 512 tokens    20 rows 15, 17   32 rows 16, 18   40 rows 24, 20
//   head_dim 64, 4 x 3 heads, 8192 tokens    20 rows 20, 19   32 rows 22, 20   40 rows 24, 20
//   head_dim 256, 2 x 2 heads, 8192 tokens   16 rows 22, 24   20 rows 29, 25   32 rows 31, 25
// (One sequence of two heads and 512 tokens would be better off with the step
// kernel even at 128 rows, 14 against 18 us; lengths are not known here.)
int chunk_min_rows(int head_dim) { return head_dim <= 128 ? 33 : 17; }

// Tokens that a tile of the tcgen05 kernel adds up at most, also where a caller
// asks for longer splits: the tensor cores truncate as they add, and a sum over n tokens comes
// out about 6e-9 n too small (measured, bf16 out, 6.5e-3 at a million tokens in one sum),
// which has to stay below what the output's rounding takes, 2^-11 (fp16) and 2^-8 (bf16) at most.
constexpr int64_t kChunkHalfTokens = 16384, kChunkBf16Tokens = 131072;

// Tokens for each CTA of a cluster up to which a cluster for each kv head of
// each sequence is taken, rather than even shares of all CTAs and a second
// launch. Measured at head_dim 128, cluster and shares in us, 4096 / 8192 /
// 16384 tokens: one sequence of 8 heads 10.8, 14.2 / 14.4, 16.1 / 21.8, 18.0;
// eight of them 16.0, 24.1 / 23.9, 30.7 / 39.7, 43.6 (head_dim 64, 3 heads:
// 8.5, 10.7 / 10.8, 12.1 / 15.6, 15.2).
constexpr int kClusterTokens = 1024;

AttnPlan plan_attention(const AkvQ4AttnDesc* d) {
    AttnPlan a = {};
    const AkvQ4Cache& c = d->cache;
    const int64_t bh = static_cast<int64_t>(c.batch) * c.kv_heads;
    a.rows = d->q_tokens * (d->q_heads / c.kv_heads);
    a.nt = c.head_dim <= 128 && a.rows > 8 ? 2 : 1;
    a.chunk = a.rows >= chunk_min_rows(c.head_dim) && d->q_dtype != AKV_Q_F32 && d->out_dtype != AKV_Q_F32;
    a.split = d->split_tokens;
    const bool shared = a.chunk && a.rows <= 128 && c.head_dim <= 128;  // its two tiles share the rows and take every other step
    const int group = a.chunk ? (c.head_dim <= 128 ? 256 : 128) : 8 * a.nt;  // rows of a CTA
    const int64_t units = bh * ((a.rows + group - 1) / group), sms = sm_count();
    size_t parts;  // rows of partials
    if (a.chunk) {
        const int64_t steps = (static_cast<int64_t>(c.max_tokens) + kChunkTokens - 1) / kChunkTokens;
        // (Two tiles that take every other step share a split.)
        const int64_t longest = (d->out_dtype == AKV_Q_F16 ? kChunkHalfTokens : kChunkBf16Tokens) * (shared ? 2 : 1);
        if (a.split == 0) {
            // One CTA per SM; the number of splits, up to eight or one wave, is
            // that of the least cost over the waves, as in the 8-bit cache. Where
            // sequences have lengths of their own and do not fill the SMs, as many
            // more as cost 15 % at most if all are full: short ones leave SMs free
            // that the long ones' splits then use. Measured, with and without, in us:
            // 32 + 8 heads, 4 x 128 of 8192 tokens, ragged 60, 85, all full 100, 86;
            // 3 x 300 of 8192 93, 133 and 165, 135; 64 + 8 heads, 8 x 5 of 8192 40, 54 and 69, 56.
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
        const int64_t chunks = units * ((c.max_tokens + q8::kShareTokens - 1) / q8::kShareTokens);
        const int64_t slots = sms * (c.head_dim > 128 || a.nt == 2 ? 2 : 4);
        a.share_min = a.split > q8::kShareTokens ? a.split / q8::kShareTokens : 1;
        const int64_t ctas = chunks / a.share_min < slots ? chunks / a.share_min : slots;
        a.share_ctas = static_cast<int>(ctas > 0 ? ctas : 1);
        a.long_sums = q8::step_sums_long(chunks, a.share_ctas, a.share_min, c.max_tokens, d->out_dtype);
        parts = 2 * static_cast<size_t>(a.share_ctas) * group;
        // The largest cluster with which all units fit the GPU at once.
        int size = q8::kStepCluster;
        while (size > 1 && bh * size > slots) size /= 2;
        a.cluster = a.split == 0 && a.rows <= 8 && c.max_tokens <= kClusterTokens * size ? size : 0;
    }
    const auto up = [](size_t x) { return (x + 15) / 16 * 16; };
    a.part_ml = 0;
    a.part_o = up(parts * sizeof(float2));
    a.bytes = a.part_o + up(parts * c.head_dim * sizeof(float)) + 16;
    return a;
}

template <int DP, bool SHARED>
int launch_chunk(const Q4Params& p, cudaStream_t s) {
    const auto kern = chunk_kernel<DP, SHARED>;
    constexpr int bytes = sizeof(ChunkSmem<DP>) + 1024;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return AKV_ERR_CUDA;
    }
    const int parts = SHARED ? p.a.nsplits / 2 : p.a.nsplits;
    constexpr int rows = 128 * kChunkTiles<DP>;
    const dim3 grid(parts * ((p.a.R + rows - 1) / rows), p.c.H, p.c.B);
    kern<<<grid, kChunkThreads<DP, SHARED>, bytes, s>>>(p);
    return q8::launched();
}

int launch_chunk(const Q4Params& p, cudaStream_t s) {
    if (p.c.D > 128) return launch_chunk<256, false>(p, s);
    if (p.a.R <= 128) return p.c.D > 64 ? launch_chunk<128, true>(p, s) : launch_chunk<64, true>(p, s);
    return p.c.D > 64 ? launch_chunk<128, false>(p, s) : launch_chunk<64, false>(p, s);
}

// Tokens from which an append's queries get a launch of their own, whose kernel
// needs fewer registers, beside the kernel with two chunks a lane and beside the
// general one. Measured with 32 + 2 x 8 heads, together and apart in us:
//   tokens                 1024       2048       4096       8192      32768
//   head_dim 128      7.2,  9.0  9.7, 11.7   20, 21     41, 38    152, 127
//   head_dim  64      5.9,  7.2  7.4,  8.7   11, 12     21, 21     81,  72
//   96, general       8.4,  8.6   13, 12     28, 20     55, 38    223, 136
//   160, general       13,  11    27, 19     52, 35    108, 70    425, 247
constexpr int64_t kQueriesApart = 8192, kQueriesApartGeneral = 2048;

// Tokens from which an append takes the kernel with two chunks a lane, where it
// can, which has longer to go before its first load. Measured likewise, the
// general kernel and that one in us, at 1 / 64 / 128 / 1024 / 32768 tokens:
// head_dim 128 2.8, 3.3 / 3.6, 3.7 / 4.4, 4.0 / 8.5, 7.2 / 154, 127; head_dim
// 256 3.0, 3.5 / 4.2, 4.2 / 4.9, 4.2 / 14, 11 / 301, 242.
constexpr int64_t kPairsTokens = 128;

template <typename T, bool VEC>
void launch_append(const AppendParams& p, int turn, dim3 grid, cudaStream_t s) {
    if (turn == kHalves) append_kernel<T, VEC, kHalves><<<grid, kAppendThreads, 0, s>>>(p);
    else if (turn == kInterleaved) append_kernel<T, VEC, kInterleaved><<<grid, kAppendThreads, 0, s>>>(p);
    else append_kernel<T, VEC, kStay><<<grid, kAppendThreads, 0, s>>>(p);
}

}  // namespace
}  // namespace q4
}  // namespace akv

using namespace akv;
using namespace akv::q4;

extern "C" {

size_t akv_q4_struct_size(int which) {
    switch (which) {
        case 0: return sizeof(AkvQ4Cache);
        case 1: return sizeof(AkvQ4AppendDesc);
        case 2: return sizeof(AkvQ4RestoreDesc);
        case 3: return sizeof(AkvQ4AttnDesc);
        default: return 0;
    }
}

int akv_q4_append(const AkvQ4AppendDesc* d, void* stream) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->cache)) return st;
    if (d->tokens < 0 || !valid_dtype(d->dtype)) return AKV_ERR_INVALID_ARGUMENT;
    const bool turn = d->rotary.table_dev, queries = d->q_dev;
    if (turn) {
        if (int st = check_rotary(d->rotary, d->cache.head_dim)) return st;
    }
    if ((queries && (!turn || d->q_heads <= 0)) || (d->positions_dev && !turn)) return AKV_ERR_INVALID_ARGUMENT;
    if (d->cache.batch == 0 || d->tokens == 0) return AKV_OK;
    const int64_t elem = size_of(d->dtype);
    if (!d->k_dev || !d->v_dev || !d->start_dev || !aligned(d->k_dev, elem) || !aligned(d->v_dev, elem) || !aligned(d->q_dev, elem) ||
        !words({d->start_dev, d->counts_dev, d->positions_dev}) || (queries && (!d->q_out_dev || !aligned(d->q_out_dev, 16))))
        return AKV_ERR_INVALID_ARGUMENT;
    AppendParams p;
    p.c = to_dev(d->cache);
    if (turn) p.r = to_dev(d->rotary);
    else p.r = RotaryDev{};
    p.x[0] = d->k_dev; p.x[1] = d->v_dev; p.x[2] = d->q_dev;
    bool vec = true;
    const int64_t* strides[3] = {d->k_stride, d->v_stride, d->q_stride};
    for (int i = 0; i < 3; ++i) {
        p.xB[i] = strides[i][0]; p.xT[i] = strides[i][1]; p.xH[i] = strides[i][2];
        if (i == 2 && !queries) break;
        vec = vec && aligned(p.x[i], 16);
        for (int k = 0; k < 3; ++k) vec = vec && strides[i][k] * elem % 16 == 0;
    }
    // No piece of eight channels is rotated in part, or has half of its other channels elsewhere.
    if (turn) vec = vec && p.r.R % (d->rotary.interleaved ? 8 : 16) == 0;
    p.q_out = d->q_out_dev;
    p.start = d->start_dev; p.counts = d->counts_dev; p.places = d->positions_dev;
    p.n = d->tokens; p.Hq = queries ? d->q_heads : 0;
    // Two chunks of eight channels a lane, where both halves of the rotated and of the other channels hold whole groups.
    const int64_t tokens = static_cast<int64_t>(p.c.B) * p.n;
    const bool pairs = vec && tokens >= kPairsTokens && (!turn || !d->rotary.interleaved) && p.r.R % 64 == 0 && (p.c.D - p.r.R) % 64 == 0;
    const int rows = 32 / (p.c.D / (pairs ? 16 : 8)) * (kAppendThreads / 32);  // tokens of a CTA
    const int64_t blocks = (tokens + rows - 1) / rows;
    if (blocks > 0x7FFFFFFF) return AKV_ERR_UNSUPPORTED;
    // As many heads a CTA as leave a wave of CTAs, in whole rounds of a lane's loads.
    const int64_t wave = 2 * static_cast<int64_t>(sm_count()), want = wave > blocks ? wave / blocks : 1;
    const auto split = [&](int heads, int round) {
        int rounds = 8 / round;
        while (rounds > 1 && (heads + rounds * round - 1) / (rounds * round) < want) --rounds;
        const int n = (heads + rounds * round - 1) / (rounds * round);
        return n < want ? static_cast<int>(want < heads ? want : heads) : n;
    };
    p.kv_splits = split(p.c.H, kAppendHeads);
    RotateParams r = {};
    r.r = p.r;
    r.B = p.c.B; r.n = p.n; r.H = p.Hq; r.D = p.c.D;
    r.x = d->q_dev; r.out = d->q_out_dev;
    r.xB = p.xB[2]; r.xT = p.xT[2]; r.xH = p.xH[2];
    r.oH = p.c.D; r.oT = r.oH * r.H; r.oB = r.oT * r.n;
    r.places = p.places; r.start = p.start; r.counts = p.counts; r.status = p.c.status;
    const bool apart = queries && tokens >= (pairs ? kQueriesApart : kQueriesApartGeneral) && rotate_fits(r, d->dtype, d->rotary.interleaved != 0);
    p.q_splits = queries && !apart ? split(p.Hq, pairs ? kRotateHeads : 2) : 0;
    if (p.kv_splits + p.q_splits > kMaxGridYZ) return AKV_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(blocks), p.kv_splits + p.q_splits);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int how = !turn ? kStay : d->rotary.interleaved ? kInterleaved : kHalves;
    with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        if (pairs) {
            if (p.q_splits) append_pairs_kernel<T, true, true><<<grid, kAppendThreads, 0, s>>>(p);
            else if (turn) append_pairs_kernel<T, true, false><<<grid, kAppendThreads, 0, s>>>(p);
            else append_pairs_kernel<T, false, false><<<grid, kAppendThreads, 0, s>>>(p);
        } else if (vec) launch_append<T, true>(p, how, grid, s);
        else launch_append<T, false>(p, how, grid, s);
    });
    if (const int st = q8::launched()) return st;
    return apart ? launch_rotate(r, d->dtype, d->rotary.interleaved != 0, s) : AKV_OK;
}

int akv_q4_restore(const AkvQ4RestoreDesc* d, void* stream) {
    if (!d) return AKV_ERR_INVALID_ARGUMENT;
    if (int st = check_cache(d->cache)) return st;
    if (d->tokens < 0 || !valid_dtype(d->dtype)) return AKV_ERR_INVALID_ARGUMENT;
    if (d->cache.batch == 0 || d->tokens == 0) return AKV_OK;
    if (!d->k_dev || !d->v_dev || !aligned(d->k_dev, 16) || !aligned(d->v_dev, 16) || !words({d->start_dev})) return AKV_ERR_INVALID_ARGUMENT;
    RestoreParams p;
    p.c = to_dev(d->cache);
    p.out[0] = d->k_dev; p.out[1] = d->v_dev;
    p.start = d->start_dev; p.n = d->tokens;
    const int64_t pieces = static_cast<int64_t>(p.n) * p.c.H * (p.c.D / 16);  // of a sequence's side
    if (pieces > 0x7FFFFF00) return AKV_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>((pieces + 255) / 256), 2 * p.c.B);
    int st = AKV_OK;
    with_type(d->dtype, [&](auto t) { st = launch_after(restore_kernel<decltype(t)>, grid, 256, static_cast<cudaStream_t>(stream), p); });
    return st;
}

size_t akv_q4_attention_workspace(const AkvQ4AttnDesc* d) { return check_attention(d) == AKV_OK ? plan_attention(d).bytes : 0; }

int akv_q4_attention(const AkvQ4AttnDesc* d, void* stream) {
    if (int st = check_attention(d)) return st;
    if (d->cache.batch == 0 || d->q_tokens == 0) return AKV_OK;
    const int64_t elem = size_of(d->q_dtype);
    if (!d->q_dev || !d->out_dev || !aligned(d->q_dev, elem) || !aligned(d->out_dev, 16)) return AKV_ERR_INVALID_ARGUMENT;
    const AttnPlan plan = plan_attention(d);
    if (!d->workspace_dev || d->workspace_bytes < plan.bytes) return AKV_ERR_WORKSPACE;
    if (!aligned(d->workspace_dev, 16)) return AKV_ERR_INVALID_ARGUMENT;
    char* ws = static_cast<char*>(d->workspace_dev);
    Q4Params pp = {};
    pp.c = to_dev(d->cache);
    pp.wait_tries = d->wait_tries ? d->wait_tries : kWaitTries;
    q8::AttnParams& p = pp.a;
    p.c.B = pp.c.B; p.c.H = pp.c.H; p.c.D = pp.c.D; p.c.T = pp.c.T; p.c.status = pp.c.status;
    p.Hq = d->q_heads; p.G = d->q_heads / d->cache.kv_heads; p.n = d->q_tokens; p.R = plan.rows;
    p.q_dtype = d->q_dtype; p.out_dtype = d->out_dtype; p.causal = d->causal;
    p.q_vec = aligned(d->q_dev, 16);
    for (int i = 0; i < 3; ++i) p.q_vec &= d->q_stride[i] * elem % 16 == 0;
    p.c2 = (d->scale > 0.f ? d->scale : 1.0f / std::sqrt(static_cast<float>(p.c.D))) * 1.4426950408889634f;
    p.q = d->q_dev; p.qB = d->q_stride[0]; p.qT = d->q_stride[1]; p.qH = d->q_stride[2];
    p.lens = d->seq_lens_dev; p.q_lens = d->q_lens_dev;
    p.split = plan.split; p.nsplits = plan.nsplits;
    p.share_ctas = plan.chunk ? 0 : plan.cluster ? -plan.cluster : plan.share_ctas; p.share_min = plan.share_min; p.row_group = 8 * plan.nt;
    p.long_sums = plan.long_sums;
    p.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
    p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
    p.out = d->out_dev; p.lse_out = d->lse_dev;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int row = pp.c.D / 2;
    const bool dense = (pp.c.D == 64 || pp.c.D == 128 || pp.c.D == 256) && pp.c.k.sT == row && pp.c.v.sT == row;
    if (int st = plan.chunk ? launch_chunk(pp, s) : dense ? launch_step_dense(pp, plan.nt, s) : launch_step_strided(pp, plan.nt, s)) return st;
    // A step kernel of one CTA leaves nothing to combine.
    if (plan.chunk ? plan.nsplits <= 1 : plan.cluster || plan.share_ctas <= 1) return AKV_OK;
    const int64_t rows = static_cast<int64_t>(p.c.B) * p.c.H * p.R;
    const int64_t pieces = plan.chunk ? plan.nsplits : plan.share_ctas / (static_cast<int64_t>(p.c.B) * p.c.H) + 1;
    const bool by_warp = pieces <= 16 && rows >= 1024;  // partials of a row: few, a warp's work
    constexpr int per = q8::kCombineThreads / 32;
    const int64_t blocks = by_warp ? (rows + per - 1) / per : rows;
    return launch_after(q8::combine_kernel, dim3(static_cast<unsigned>(blocks)), q8::kCombineThreads, s, p, static_cast<int>(rows), by_warp, 0, 0, 0);
}

}  // extern "C"
