/*
 * akv_q8.h — C ABI of the 8-bit KV cache: store, attention with the weight
 * each cached token received, eviction by that weight, restore.
 *
 * A cache holds K and V as 8-bit codes with one fp32 scale for every block of
 * `block_tokens` tokens of a (sequence, kv head): value = code * scale, codes
 * int8 in [-127, 127] or e4m3. The conventions are those of akv_cuda.h:
 * caller-owned buffers, int status, stream order, no allocation, no
 * synchronisation. No call needs akv_cuda_init.
 * The reference project has no counterpart to these calls.
 */
#ifndef AKV_Q8_H
#define AKV_Q8_H

#include "akv_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AKV_Q8_INT8 0
#define AKV_Q8_E4M3 1

/*
 * K or V of a cache. Token t of (batch b, kv head h) is row t % page_tokens of
 * logical page t / page_tokens, physical page `phys` (the block table's entry,
 * or the logical page without a table); its head_dim codes start at
 *     codes + b*stride_batch + h*stride_head + phys*stride_page + row*stride_token
 * and its scale is
 *     scales[b*scale_stride_batch + h*scale_stride_head + phys*scale_stride_page
 *            + row / block_tokens].
 * Code strides are bytes and multiples of 16, codes 16-byte aligned; scale
 * strides are elements. All page_tokens rows of a page are the cache's own
 * memory (an eviction writes whole blocks). Scales are >= 0; a scale below 2^-90 counts as 2^-90
 * where V's softmax weights are formed. A NaN scale makes NaN of what sees a
 * token of its block. Codes are numbers: an e4m3 NaN code, which no call here
 * writes, may also show in queries that end before its token.
 */
typedef struct AkvQ8Side {
    void* codes;
    float* scales;
    int64_t stride_batch, stride_head, stride_page, stride_token;
    int64_t scale_stride_batch, scale_stride_head, scale_stride_page;
} AkvQ8Side;

typedef struct AkvQ8Cache {
    int32_t format;                 /* AKV_Q8_* */
    int32_t block_tokens;           /* tokens per scale: 16, 32, 64 or 128 */
    int32_t batch, kv_heads, head_dim; /* head_dim a multiple of 16, at most 256 */
    int32_t max_tokens;             /* tokens per sequence the cache has room for */
    int32_t page_tokens;            /* multiple of block_tokens */
    int32_t pages_per_seq, num_pages; /* of the block table */
    int32_t reserved0;
    const int32_t* block_table_dev; /* [batch][pages_per_seq] or NULL */
    AkvQ8Side k, v;
    int32_t* status_dev;            /* optional: kernels write AKV_ERR_BAD_BLOCK_TABLE (an entry outside
                                       [0, num_pages): reads as zeros, writes are dropped) or
                                       AKV_ERR_INVALID_ARGUMENT (a store outside [0, max_tokens)) here, or
                                       AKV_ERR_TIMEOUT (a bounded wait inside a kernel ran out: its rows are NaN) */
} AkvQ8Cache;

/*
 * Store tokens: rows i < counts[b] (n without counts) of k/v
 * [batch][n][kv_heads][head_dim], element strides batch / token / head in
 * k_stride / v_stride, go to tokens start[b] + i. Each touched block gets
 * scale = amax * (1/127) (1/448 for e4m3) over its new rows and
 * code = round_half_even(x * (1/scale)); a block that holds rows before
 * start[b] keeps its scale unless the new rows need a larger one, and then
 * its rows are rounded again under that one. Tokens are stored in order: what
 * a block holds from start[b] on is not kept. A block that is given an
 * infinity or a NaN gets a NaN scale and codes of 0; one whose scale would be
 * subnormal is stored as zeros. Rows past max_tokens are dropped, with a start
 * outside [0, max_tokens) all rows of the sequence (see status_dev).
 */
typedef struct AkvQ8StoreDesc {
    AkvQ8Cache cache;
    int32_t tokens;                 /* n */
    int32_t dtype;                  /* AKV_Q_* */
    const void* k_dev;
    const void* v_dev;
    int64_t k_stride[3], v_stride[3];
    const int32_t* start_dev;       /* [batch] */
    const int32_t* counts_dev;      /* [batch] or NULL */
} AkvQ8StoreDesc;

int akv_q8_store(const AkvQ8StoreDesc* desc, void* stream);

/*
 * Restore: token start[b] + i (0 without start), i < tokens, of every head as
 * k/v [batch][tokens][kv_heads][head_dim] of `dtype`, code * scale rounded
 * once. Tokens outside [0, max_tokens) give zeros.
 */
typedef struct AkvQ8RestoreDesc {
    AkvQ8Cache cache;
    int32_t tokens;
    int32_t dtype;                  /* AKV_Q_* */
    const int32_t* start_dev;       /* [batch] or NULL */
    void* k_dev;
    void* v_dev;
} AkvQ8RestoreDesc;

int akv_q8_restore(const AkvQ8RestoreDesc* desc, void* stream);

/*
 * Attention of q_tokens query tokens per sequence over its first seq_lens[b]
 * cached tokens, kv head = query head / (q_heads / kv_heads). The queries are
 * the sequence's newest tokens (their K and V are stored already): with
 * `causal`, query i of q_lens[b] (q_tokens without q_lens) sees tokens
 * t <= seq_lens[b] - q_lens[b] + i, without it all of them.
 *     out = softmax(scale q.K) V,  lse = ln sum exp(scale q.K),
 *     weights[b][h][t] (+)= sum over queries and query heads of h of the
 *                           softmax weight of t   (accumulate 1: +=, 0: =)
 * A query that sees nothing, and one past q_lens[b], gives zeros and
 * lse = -inf. With accumulate 0 the weights of tokens past seq_lens[b] become
 * 0, with 1 they stay.
 *
 * Scores, softmax and sums are fp32. A score is a sum in the tensor cores,
 * which truncate, of exact products (of 22 bits with fp32 queries): off by at
 * most 2^-20 of the sum of |scale q K|. With an fp32 output the softmax weights
 * meet V in two fp16 parts (22 bits) and long sums are rounded to nearest
 * every 32 products; with a 16-bit output the weights are rounded to fp16,
 * and from 33 rows (queries x heads of a kv head; 17 above head_dim 128)
 * the values' sum comes out 6e-9 of itself per token of a split too small.
 *
 * Lengths are read by the kernels, so what the host decides, the splits of many
 * rows and the size of the workspace, goes by max_tokens: a cache with much
 * more room than tokens is served best through one with a smaller max_tokens
 * over the same memory. Workspace: partials, and with weights of up to 16 rows
 * (8 above head_dim 128) 4 bytes per row, kv head and token of max_tokens.
 */
typedef struct AkvQ8AttnDesc {
    AkvQ8Cache cache;
    int32_t q_heads, q_tokens;
    int32_t q_dtype, out_dtype;     /* AKV_Q_* */
    int32_t causal, accumulate;
    int32_t split_tokens;           /* tokens per split at least, a multiple of 16; 0 = library choice */
    float scale;                    /* 0 = head_dim^-0.5 */
    const void* q_dev;              /* element strides batch / token / head */
    int64_t q_stride[3];
    const int32_t* seq_lens_dev;    /* [batch] or NULL (= max_tokens) */
    const int32_t* q_lens_dev;      /* [batch] or NULL (= q_tokens) */
    void* out_dev;                  /* [batch][q_tokens][q_heads][head_dim] */
    float* lse_dev;                 /* [batch][q_tokens][q_heads] or NULL */
    float* weights_dev;             /* [batch][kv_heads], rows weights_stride apart, or NULL */
    int64_t weights_stride;
    void* workspace_dev;            /* 16-byte aligned, see akv_q8_attention_workspace */
    size_t workspace_bytes;
} AkvQ8AttnDesc;

/* Workspace bytes of a descriptor (at least 16); 0 for one that would be refused. */
size_t akv_q8_attention_workspace(const AkvQ8AttnDesc* desc);
int akv_q8_attention(const AkvQ8AttnDesc* desc, void* stream);

/*
 * Evict: each kv head of each sequence keeps min(len, keep) of its len =
 * seq_lens[b] tokens. When len > keep these are the first `sinks`, the last
 * `recent` and, of the others, those of the largest weights[b][h][t] (equal
 * weights: the lower index; a NaN ranks highest). They are packed in their
 * order into `dst`, a cache in other memory with the same format, batch,
 * kv_heads and head_dim, whose blocks get scales of their own (as a store
 * of the restored rows would); its rows from min(len, keep) to the end of
 * their block become zeros. Other memory are also other pages of the same
 * pool: no page of dst's table may be in src's, which the call cannot see.
 *     kept[b][h][i]        token that row i was, -1 from min(len, keep) on
 *     out_lens[b]          min(len, keep)
 *     out_weights[b][h][i] its weight, 0 from min(len, keep) up to
 *                          out_weights_tokens: dst.max_tokens there leaves no
 *                          earlier tokens' weights where later ones will be
 */
typedef struct AkvQ8EvictDesc {
    AkvQ8Cache src, dst;
    const float* weights_dev;       /* [batch][kv_heads], rows weights_stride apart */
    int64_t weights_stride;
    const int32_t* seq_lens_dev;    /* [batch] or NULL (= src.max_tokens) */
    int32_t keep, sinks, recent;    /* sinks + recent <= keep <= dst.max_tokens */
    int32_t out_weights_tokens;     /* weights written per row, keep to out_weights_stride; 0 = keep */
    int32_t* kept_dev;              /* [batch][kv_heads][keep] */
    int32_t* out_lens_dev;          /* [batch] */
    float* out_weights_dev;         /* [batch][kv_heads], rows out_weights_stride apart (>= keep) */
    int64_t out_weights_stride;
} AkvQ8EvictDesc;

int akv_q8_evict(const AkvQ8EvictDesc* desc, void* stream);

/* Host-only: sizeof of AkvQ8Cache (0), AkvQ8StoreDesc (1), AkvQ8RestoreDesc
 * (2), AkvQ8AttnDesc (3), AkvQ8EvictDesc (4); 0 otherwise. */
size_t akv_q8_struct_size(int which);

#ifdef __cplusplus
}
#endif

#endif /* AKV_Q8_H */
