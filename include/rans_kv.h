/*
 * rans_kv.h -- C ABI of the paged key-value cache of librans_b200.so: the part
 * of a decoder step between the v and the o projection.  Plain pointers, sizes
 * and an int status.
 *
 * A cache holds `pages` pages of `page` token slots for each of `kv_heads`
 * heads.  Sequence b (0..batch-1) owns the pages table[b * table_cols + i]; its
 * token in place t (0..length[b]-1) lies in slot t % page of its page t / page.
 * Rows of keys and values are `dim` bf16 or fp16 values, or 4-bit rows:
 *
 *   blocks of 32 values x with one scale 2^e, e = clamp(floor(log2 max|x|) - 2,
 *   -63, 63), stored as the byte e + 127 (255 when the block holds a value that
 *   is not finite: the whole block then reads as NaN, whatever its codes; other
 *   bytes than 64..190 and 255 do not occur); each value as the e2m1 code
 *   (sign, two exponent bits, one fraction bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6)
 *   nearest to x / 2^e, ties to the even code, at most 6.  A row is dim/2 bytes
 *   of codes and, in arrays of their own, dim/32 scale bytes.  Value d, of block
 *   n = d / 32, lies in byte (d % 32 / 8) * dim/8 + 4 n + d % 8 / 2, in the low
 *   half when d is even: the dim/8 bytes from (d % 32 / 8) * dim/8 hold a quarter
 *   of every block, which is what one thread of the attention multiplies.
 *
 * All launchers are asynchronous on `stream`, allocate nothing, never wait for
 * another block, and return 0, a CUDA error code (as int) after a failed
 * launch, -1 for an unsupported kind or dim, -2 for bad shapes, pointers or
 * alignment, -3 when the workspace is too small.  A page number outside
 * 0..pages-1 or a length beyond the table is never followed: the token is left
 * out and a bit of *status is raised (RANS_KV_BAD_PAGE, RANS_KV_BAD_LENGTH).
 * Rows outside `starts` and starts beyond the rows are left out and not counted;
 * where starts fall, append adds nothing (RANS_KV_BAD_STARTS in each case).
 * Pages may be shared by sequences for attention alone; append, weigh and evict
 * want each page in one place of the table.
 * Calls on one cache share its workspace and books and have to be ordered (one
 * stream, or events between streams).  No counterpart in the reference, which
 * stops at the weight products (kernel/bench.py:104-107).
 */
#ifndef RANS_KV_H
#define RANS_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef __CUDA_RUNTIME_H__
typedef struct CUstream_st* cudaStream_t;
#endif

enum { RANS_KV_BF16 = 0, RANS_KV_FP16 = 1, RANS_KV_MXFP4 = 2, RANS_KV_FP32 = 3 };
enum { RANS_KV_BAD_PAGE = 1, RANS_KV_BAD_LENGTH = 2, RANS_KV_BAD_STARTS = 4 };

#define RANS_KV_MAX_BATCH 2048

/* One cache.  Device pointers.  Strides are in bytes, multiples of 16, and the
 * bases are 16-byte aligned (bf16, fp16); 4-bit rows, scales, weight and
 * position are contiguous [pages][kv_heads][page][...] arrays (k_page .. v_slot
 * are ignored then). */
typedef struct RansKvCache {
    void* k;
    void* v;
    uint8_t* k_scale;            /* 4-bit rows only, else NULL                    */
    uint8_t* v_scale;
    float* weight;               /* attention weight each token received, or NULL */
    int32_t* position;           /* place of each token in its sequence, or NULL  */
    const int32_t* table;        /* [batch][table_cols]                           */
    int32_t* length;             /* [batch] tokens in the cache                   */
    int32_t* seen;               /* [batch] tokens appended so far                */
    int32_t* status;             /* one word, bits RANS_KV_BAD_*                  */
    void* workspace;             /* its first rans_kv_counter_bytes are zero      */
    int64_t workspace_bytes;     /* before the first call and stay zero after     */
    int64_t k_page, k_head, k_slot;
    int64_t v_page, v_head, v_slot;
    int32_t pages, page;         /* page: a multiple of 16                        */
    int32_t kv_heads, dim;       /* dim: 64, 128 or 256                           */
    int32_t batch, table_cols;
    int32_t kind;                /* RANS_KV_BF16, _FP16 or _MXFP4                 */
    int32_t reserved;            /* must be 0                                     */
} RansKvCache;

/* Leading workspace bytes that have to be zero before the first call. */
int64_t rans_kv_counter_bytes(const RansKvCache* c);

/* Workspace bytes for attention with `heads` query heads (weigh: also the
 * accumulation of weights), and for eviction to `budget` tokens. */
int64_t rans_kv_attend_bytes(const RansKvCache* c, int heads, int weigh);
int64_t rans_kv_evict_bytes(const RansKvCache* c, int budget);

/* Append `tokens` rows to the sequences: k and v are [tokens][kv_heads][dim] of
 * type `given` (RANS_KV_BF16, _FP16 or _FP32) with byte strides per token and
 * head (multiples of 16, bases 16-byte aligned).  Sequence b gets the rows
 * starts[b]..starts[b+1]-1 (device int32[batch+1], rising from 0 to tokens), or
 * with starts NULL row b (tokens == batch).  Values are rounded to the cache's
 * type; position becomes seen[b] + i, weight 0; length and seen grow. */
int rans_kv_append(const RansKvCache* c, const void* k, const void* v, int given,
                   int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                   const int32_t* starts, int tokens, cudaStream_t stream);

/* The last starts[b+1]-starts[b] tokens of every sequence back as contiguous
 * rows k_out, v_out [tokens][kv_heads][dim] (fp16 for an fp16 cache, else bf16:
 * every 4-bit value is exact in it). */
int rans_kv_read(const RansKvCache* c, void* k_out, void* v_out, const int32_t* starts, int tokens,
                 cudaStream_t stream);

/* Attention of one query per sequence over its length[b] tokens:
 *   s_t = scale * q . k_t,  out = sum_t exp(s_t) v_t / sum_t exp(s_t),
 *   log_sum = log sum_t exp(s_t)
 * for q [batch][heads][dim] of type `q_kind` (the cache's type; bf16 or fp16 over
 * 4-bit rows), byte strides per sequence and head; query head i reads kv head
 * i / (heads / kv_heads).  out has q's type, contiguous like log_sum (fp32
 * [batch][heads], may be NULL).  A sequence without tokens gets zeros and
 * -infinity.  weigh != 0 also adds sum over a kv head's query heads of
 * exp(s_t - log_sum) to the cache's weight of every token, in one fixed order. */
int rans_kv_attend(const RansKvCache* c, const void* q, int q_kind, int64_t q_batch, int64_t q_head, int heads,
                   float scale, void* out, float* log_sum, int weigh, cudaStream_t stream);

/* Bring every sequence with more than `budget` tokens back to `budget`, per kv
 * head: the `recent` newest tokens (position >= seen[b] - recent) and the
 * heaviest others stay (ties: the lower place; NaN counts as heaviest).  The
 * i-th kept token at or above place `budget` moves, with its position and
 * weight, into the i-th freed place below it; nothing else moves. */
int rans_kv_evict(const RansKvCache* c, int budget, int recent, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* RANS_KV_H */
