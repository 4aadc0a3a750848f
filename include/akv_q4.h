/*
 * akv_q4.h — C ABI of the 4-bit KV cache: append with the position rotation on
 * the way, attention, restore.
 *
 * A cache holds K and V as e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign),
 * two a byte, with an fp16 scale for every 32 channels of a token:
 * value = code * scale, rounded to fp16. 4.5 bits a value. Since no scale
 * spans tokens, an append only writes.
 * Conventions of akv_cuda.h: caller-owned buffers, int status, stream order,
 * no allocation, no synchronisation. No call needs akv_cuda_init.
 * The reference project has no counterpart to these calls.
 */
#ifndef AKV_Q4_H
#define AKV_Q4_H

#include "akv_rotary.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AKV_Q4_GROUP 32             /* channels of a scale */
#define AKV_Q4_TOKENS 16            /* pages hold a multiple of so many tokens */

/*
 * K or V of a cache. Token t of (batch b, kv head h) is row t % page_tokens of
 * logical page t / page_tokens, physical page `phys` (the block table's entry,
 * or the logical page without a table). Its head_dim codes are the bytes at
 *     codes + b*stride_batch + h*stride_head + phys*stride_page + row*stride_token,
 * channel 2i in the lower half of byte i, sign in a code's top bit; the scale
 * of its channels 32 g to 32 g + 31 is
 *     scales[b*scale_stride_batch + h*scale_stride_head + phys*scale_stride_page
 *            + g*scale_stride_group + row].
 * Code strides are bytes and multiples of 16, codes 16-byte aligned; scale
 * strides are elements and multiples of 4, scales 8-byte aligned. All rows of
 * a page (a multiple of AKV_Q4_TOKENS) are the cache's own memory, in the
 * scales too. Scales are >= 0. A token with NaN in K's scales makes NaN of
 * every query that sees it and of no other. V's scales are numbers: an
 * infinity or a NaN there, which no call here writes, may also show in queries
 * that end before its token.
 */
typedef struct AkvQ4Side {
    void* codes;
    void* scales;                   /* fp16 */
    int64_t stride_batch, stride_head, stride_page, stride_token;
    int64_t scale_stride_batch, scale_stride_head, scale_stride_page, scale_stride_group;
} AkvQ4Side;

typedef struct AkvQ4Cache {
    int32_t batch, kv_heads, head_dim; /* head_dim a multiple of 32, at most 256 */
    int32_t max_tokens;             /* tokens per sequence the cache has room for */
    int32_t page_tokens;            /* multiple of AKV_Q4_TOKENS */
    int32_t pages_per_seq, num_pages; /* of the block table */
    int32_t reserved0;
    const int32_t* block_table_dev; /* [batch][pages_per_seq] or NULL */
    AkvQ4Side k, v;
    int32_t* status_dev;            /* optional: kernels write AKV_ERR_BAD_BLOCK_TABLE (an entry outside
                                       [0, num_pages): reads as zeros, writes are dropped),
                                       AKV_ERR_INVALID_ARGUMENT (an append outside [0, max_tokens) or a position
                                       outside the table) or AKV_ERR_TIMEOUT (a bounded wait inside a kernel ran
                                       out: its rows are NaN) here */
} AkvQ4Cache;

/*
 * Append: rows i < counts[b] (n without counts) of k/v
 * [batch][n][kv_heads][head_dim], element strides batch / token / head, become
 * tokens start[b] + i. With a rotary table (table_dev not NULL) k is rotated
 * first, as akv_rotate does but without rounding to `dtype`, at
 * positions[axis][b][i], or start[b] + i on every axis without positions.
 * Then, for each 32 channels of a token,
 *     scale = min(fp16(amax * (1/6)), 10912), code = e2m1(x / scale),
 * product and quotient (and 1/6) rounded to fp32, then to fp16 and e2m1, to the
 * nearest (ties to even), codes beyond 6 to 6; with a scale of 0 the codes are 0. (Values beyond 65472
 * become 65472.) A token whose K or V row holds an infinity or a NaN gets NaN
 * as K's scales and 0 as K's codes; V's groups that hold one become 0. The
 * same where a position is outside the table. Rows past max_tokens are
 * dropped, with a start outside [0, max_tokens) all rows of the sequence (see
 * status_dev).
 * With q [batch][n][q_heads][head_dim] the queries of the same tokens are
 * rotated (a table is needed) to q_out, contiguous: rounded once to `dtype`,
 * zeros past counts[b].
 */
typedef struct AkvQ4AppendDesc {
    AkvQ4Cache cache;
    AkvRotary rotary;               /* table_dev NULL: no rotation */
    int32_t tokens;                 /* n */
    int32_t dtype;                  /* AKV_Q_*, of k, v, q and q_out */
    int32_t q_heads, reserved0;
    const void* k_dev;
    const void* v_dev;
    const void* q_dev;              /* or NULL */
    void* q_out_dev;
    int64_t k_stride[3], v_stride[3], q_stride[3];
    const int32_t* start_dev;       /* [batch] */
    const int32_t* counts_dev;      /* [batch] or NULL */
    const int32_t* positions_dev;   /* [axes][batch][n] or NULL */
} AkvQ4AppendDesc;

int akv_q4_append(const AkvQ4AppendDesc* desc, void* stream);

/*
 * Restore: token start[b] + i (0 without start), i < tokens, of every head as
 * k/v [batch][tokens][kv_heads][head_dim] of `dtype`. Tokens outside
 * [0, max_tokens) give zeros.
 */
typedef struct AkvQ4RestoreDesc {
    AkvQ4Cache cache;
    int32_t tokens;
    int32_t dtype;                  /* AKV_Q_* */
    const int32_t* start_dev;       /* [batch] or NULL */
    void* k_dev;
    void* v_dev;
} AkvQ4RestoreDesc;

int akv_q4_restore(const AkvQ4RestoreDesc* desc, void* stream);

/*
 * Attention of q_tokens query tokens per sequence over its first seq_lens[b]
 * cached tokens, kv head = query head / (q_heads / kv_heads). The queries are
 * the sequence's newest tokens (appended already): with `causal`, query i of
 * q_lens[b] (q_tokens without q_lens) sees tokens
 * t <= seq_lens[b] - q_lens[b] + i, without it all of them.
 *     out = softmax(scale q.K) V,  lse = ln sum exp(scale q.K)
 * A query that sees nothing, and one past q_lens[b], gives zeros and lse = -inf.
 *
 * Scores, softmax and sums are fp32. A score is a sum in the tensor cores,
 * which truncate, of exact products (of 22 bits with fp32 queries): off by at
 * most 2^-20 of the sum of |scale q K|. With an fp32 output the softmax weights
 * meet V in two fp16 parts (22 bits) and long sums are rounded to nearest
 * every 32 products; with a 16-bit output the weights are rounded to fp16, and
 * the values' sum loses about 6e-9 of itself per token that the tensor cores
 * add up, never more than 16384 tokens with an fp16 output and 131072 with a
 * bf16 one; such sums are added in fp32.
 *
 * Lengths are read by the kernels, so what the host decides, the splits of many
 * rows and the size of the workspace, goes by max_tokens: a cache with much
 * more room than tokens is served best through one with a smaller max_tokens
 * over the same memory.
 */
typedef struct AkvQ4AttnDesc {
    AkvQ4Cache cache;
    int32_t q_heads, q_tokens;
    int32_t q_dtype, out_dtype;     /* AKV_Q_* */
    int32_t causal;
    int32_t split_tokens;           /* tokens per split at least (many rows and a 16-bit output: up to what a sum may
                                       hold, see above), a multiple of 16; 0 = library choice */
    float scale;                    /* 0 = head_dim^-0.5 */
    int32_t wait_tries;             /* tries, of about 4.5 us, of a wait inside a kernel before it gives up (status_dev);
                                       0 = library choice, some 19 s */
    const void* q_dev;              /* element strides batch / token / head */
    int64_t q_stride[3];
    const int32_t* seq_lens_dev;    /* [batch] or NULL (= max_tokens) */
    const int32_t* q_lens_dev;      /* [batch] or NULL (= q_tokens) */
    void* out_dev;                  /* [batch][q_tokens][q_heads][head_dim] */
    float* lse_dev;                 /* [batch][q_tokens][q_heads] or NULL */
    void* workspace_dev;            /* 16-byte aligned, see akv_q4_attention_workspace */
    size_t workspace_bytes;
} AkvQ4AttnDesc;

/* Workspace bytes of a descriptor (at least 16); 0 for one that would be refused. */
size_t akv_q4_attention_workspace(const AkvQ4AttnDesc* desc);
int akv_q4_attention(const AkvQ4AttnDesc* desc, void* stream);

/* Host-only: sizeof of AkvQ4Cache (0), AkvQ4AppendDesc (1), AkvQ4RestoreDesc
 * (2), AkvQ4AttnDesc (3); 0 otherwise. */
size_t akv_q4_struct_size(int which);

#ifdef __cplusplus
}
#endif

#endif /* AKV_Q4_H */
