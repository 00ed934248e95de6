/*
 * hbfsim/kv_v1.h -- operators over a paged key/value cache held in 8 bits
 * (additive, versioned).  They run the attention side of a decode step on
 * the GPU and say which blocks of the cache it read, so that a front end can
 * time those reads (hbfsim_submit_access_batch_v1) or place the blocks
 * (hbfsim_submit_capacity_batch_v1) instead of a synthetic trace.
 *
 * A cache is `pages` pages of `block_tokens` tokens.  For every page p and
 * key/value head h:
 *
 *   data   [pages][kv_heads][2][block_tokens][head_dim]  e4m3: the keys of
 *          the block, then its values.  With 16 tokens of 128 channels the
 *          two are 4096 contiguous bytes.
 *   scale  [pages][kv_heads][2]  fp32 powers of two: a stored value x stands
 *          for x * scale.
 *   bounds [pages][kv_heads][2][head_dim]  int8: least and greatest stored
 *          key value per channel over the tokens in use, rounded outwards to
 *          multiples of 4 and divided by 4.
 *
 * A block table (int32 [seqs][width], row stride table_stride) maps block j
 * of a sequence (tokens j*block_tokens ..) to its page.  An entry outside
 * [0, pages) is a block that is not there: its tokens are dropped by an
 * append and not seen by a query, and it is never listed.  A sequence length
 * is read as if clamped to [0, width * block_tokens].
 *
 * All pointers are device pointers.  The calls are asynchronous on `stream`
 * (a cudaStream_t; NULL is the legacy default stream), allocate nothing, and
 * return an hbfsim_error; they can be captured in a CUDA graph.  A call with
 * no work returns HBFSIM_OK and launches nothing.  Results do not depend on
 * the order in which thread blocks run.
 *
 * Limits, beyond which a call returns HBFSIM_INVALID_ARGUMENT: 2^31 - 1 pages,
 * 1024 key/value heads, 65536 sequences, 2^24 blocks and 2^31 - 1 tokens to a
 * table's row, 2^31 - 1 query rows (sequences * tokens * heads), 2^22 tokens to
 * an append.
 *
 * How a call is spread over the device follows from what the host knows: the
 * table's width and the room of the lists, not the lengths, which the device
 * reads.  A table much wider than its longest sequence takes the form for long
 * rows (one of 301 tokens then takes two kernels, 10 us, instead of one, 7 us):
 * where the lengths are known to be short, pass a smaller width with the same
 * table_stride.
 */
#ifndef HBFSIM_KV_V1_H
#define HBFSIM_KV_V1_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum hbfsim_kv_type {
    HBFSIM_KV_BF16 = 0,
    HBFSIM_KV_F16 = 1
};

#define HBFSIM_KV_V1_VERSION 1u

/* head_dim: 64, 128 or 256; block_tokens: 16, 32 or 64 (others:
 * HBFSIM_UNSUPPORTED).  data and bounds 16-byte aligned, scale 8-byte. */
typedef struct hbfsim_kv_cache_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t block_tokens;
    uint32_t reserved;
    uint64_t pages;
    void* data;
    float* scale;
    int8_t* bounds;
} hbfsim_kv_cache_v1;

/* New tokens: token i of the batch has keys k[i*k_stride_token +
 * h*k_stride_head + d] (strides in elements), values likewise.  Sequence s
 * gets tokens [offsets[s], offsets[s+1]) at positions start[s]..; offsets
 * NULL: tokens / seqs of them each.
 *
 * Per touched block, head and side (keys, values): a = largest finite |x|
 * of the new tokens, e = least integer in [-100, 120] with a <= 448 * 2^e
 * (-100 for a = 0), scale = 2^e, or the block's scale if that is larger and
 * the block holds earlier tokens (positions before start).  New values are
 * stored as x / scale rounded to e4m3 (nearest, ties to even, saturating;
 * NaN stays NaN), earlier ones are rounded again if the scale grew, slots
 * after the last new token become 0, and the bounds are taken over the
 * tokens in use (NaN counts as 0).  Positions past the table are dropped.
 * Two sequences that write one page in one call race. */
typedef struct hbfsim_kv_append_batch_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t type;               /* hbfsim_kv_type of k and v */
    uint32_t seqs;
    uint32_t width;
    uint32_t reserved;
    uint64_t tokens;
    const void* k;
    const void* v;
    int64_t k_stride_token;
    int64_t k_stride_head;
    int64_t v_stride_token;
    int64_t v_stride_head;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* start;
    const int32_t* offsets;
} hbfsim_kv_append_batch_v1;

int hbfsim_kv_append_v1(const hbfsim_kv_cache_v1* cache,
                        const hbfsim_kv_append_batch_v1* batch, void* stream);

/* Queries: the newest `tokens` tokens of every sequence (at most 16);
 * lengths counts them.  Token t of sequence s is at position
 * lengths[s] - tokens + t and sees positions up to its own. */
typedef struct hbfsim_kv_query_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t type;               /* hbfsim_kv_type of q and out */
    uint32_t seqs;
    uint32_t tokens;
    uint32_t q_heads;            /* a multiple of kv_heads, at most 64 times */
    uint32_t width;
    uint32_t reserved;
    const void* q;               /* last axis contiguous, strides in elements */
    int64_t q_stride_seq;
    int64_t q_stride_token;
    int64_t q_stride_head;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
} hbfsim_kv_query_v1;

/* Block lists by a cheap score.  The queries of a group (the query heads of
 * one key/value head) become whole numbers, qi = rint(q * 2^(7-x)) within
 * +-127, x the binary exponent of their largest magnitude; block j scores
 * (float)(sum_d sum_g max(qi, 0) * hi + min(qi, 0) * lo) * key scale, which,
 * up to the rounding of the queries, bounds the group's summed products from
 * above.  The sums are whole numbers, so lists are equal however they are
 * computed.  The first `sink` blocks and the last `recent` of what the token
 * sees are always listed, then the greatest scores, the lowest index among
 * equals.
 * blocks: int32 [seqs][tokens][kv_heads][top], ascending, -1 behind the
 * count; counts: int32 [seqs][tokens][kv_heads].  sink + recent <= top,
 * recent >= 1.  Elements of q that are not finite count as 0. */
uint64_t hbfsim_kv_select_workspace_v1(const hbfsim_kv_cache_v1* cache,
                                       const hbfsim_kv_query_v1* query);
int hbfsim_kv_select_v1(const hbfsim_kv_cache_v1* cache,
                        const hbfsim_kv_query_v1* query, uint32_t top,
                        uint32_t sink, uint32_t recent, int32_t* blocks,
                        int32_t* counts, void* workspace,
                        uint64_t workspace_bytes, void* stream);

/* Attention.  blocks NULL: over every block of the sequence; else over the
 * listed ones (int32 [seqs][tokens][kv_heads][top], the first counts[...] of
 * each list, in any order and without repetition; an index that the sequence
 * does not have is passed over).
 * out: type, [seqs][tokens][q_heads][head_dim], 4-byte aligned; a token that
 * sees nothing gets 0.  lse (NULL to skip): fp32 [seqs][tokens][q_heads], natural
 * logarithm of the sum of exponentials, -inf for such a token.  weights
 * (NULL to skip): fp32 [seqs][kv_heads][width], softmax weight of each
 * block summed over the group's heads and the tokens, every entry written. */
typedef struct hbfsim_kv_attention_args_v1 {
    uint32_t struct_size;
    uint32_t version;
    float softmax_scale;
    uint32_t top;
    const int32_t* blocks;
    const int32_t* counts;
    void* out;
    float* lse;
    float* weights;
    void* workspace;
    uint64_t workspace_bytes;
} hbfsim_kv_attention_args_v1;

uint64_t hbfsim_kv_attention_workspace_v1(const hbfsim_kv_cache_v1* cache,
                                          const hbfsim_kv_query_v1* query,
                                          const hbfsim_kv_attention_args_v1* args);
int hbfsim_kv_attention_v1(const hbfsim_kv_cache_v1* cache,
                           const hbfsim_kv_query_v1* query,
                           const hbfsim_kv_attention_args_v1* args, void* stream);

/* Eviction by accumulated attention weight.  For every block of a sequence
 *   score' = score - (score >> decay) + sum_h rint(w * 2^30)
 * (whole numbers; decay 0: no decay; w clamped to [0, 2^20], NaN as 0).  A
 * sequence of more than `keep` blocks loses those of least score', the
 * lowest index among equals, never the first `sink` nor the last `recent`
 * (sink + recent <= keep, recent >= 1, so that the block being filled
 * stays).  The others close up in order.  Table entries are carried along as
 * they are.
 * Out (in memory apart from the inputs' and from each other's): score, table
 * (rows of `width`, 0 and -1 behind the last block), lengths (less the evicted
 * blocks' tokens), freed (the evicted blocks' table entries in block order, -1
 * behind), freed_counts. */
typedef struct hbfsim_kv_evict_batch_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t seqs;
    uint32_t kv_heads;
    uint32_t width;
    uint32_t block_tokens;
    uint32_t keep;
    uint32_t sink;
    uint32_t recent;
    uint32_t decay;              /* at most 63 */
    const int64_t* score;        /* [seqs][width] */
    const float* weights;        /* [seqs][kv_heads][width] */
    const int32_t* table;        /* row stride table_stride */
    int64_t table_stride;
    const int32_t* lengths;
    int64_t* score_out;
    int32_t* table_out;
    int32_t* lengths_out;
    int32_t* freed;
    int32_t* freed_counts;
} hbfsim_kv_evict_batch_v1;

int hbfsim_kv_evict_v1(const hbfsim_kv_evict_batch_v1* batch, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HBFSIM_KV_V1_H */
