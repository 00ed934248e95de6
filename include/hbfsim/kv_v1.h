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

/* An append whose keys are turned by their positions on the way into the
 * cache, and the queries of the same tokens with them.
 *
 * A head's first 2 * pairs channels form pairs: channel i with i + pairs, or
 * with `neighbours` 2i with 2i + 1.  Pair i of token t turns by the angle
 *   a = positions[axis[i]][t] * freq[i]      (rounded to 64 bits)
 * with cos a and sin a rounded to 32 bits:
 *   (x, y) -> (x cos a - y sin a, x sin a + y cos a)
 * every product and sum rounded to 32 bits; other channels stay.  Queries are
 * rounded once, to the batch's type; keys go on in 32 bits as the new values of
 * the append above.  Values are not turned.  Every row of q is turned, rows
 * that belong to no sequence too.
 * axes: 1 to 4 (a text's one, or time, height and width); an axis of a pair
 * past them is read as the last.  pairs: a multiple of head_dim / 32, at most
 * head_dim / 2.  q_heads 0: keys alone.  q_out: the batch's type, [tokens]
 * [q_heads][head_dim], 16-byte aligned, in memory apart from the inputs' and
 * the cache's (from an input's lowest row to its highest). */
typedef struct hbfsim_kv_rotary_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t q_heads;            /* at most 65536 */
    uint32_t axes;
    uint32_t pairs;
    uint32_t neighbours;         /* 0 or 1 */
    const void* q;               /* last axis contiguous, strides in elements */
    int64_t q_stride_token;
    int64_t q_stride_head;
    void* q_out;
    const int32_t* positions;    /* [axes][tokens], rows positions_stride apart */
    int64_t positions_stride;
    const double* freq;          /* [pairs] */
    const uint8_t* axis;         /* [pairs] */
} hbfsim_kv_rotary_v1;

int hbfsim_kv_append_rotary_v1(const hbfsim_kv_cache_v1* cache,
                               const hbfsim_kv_append_batch_v1* batch,
                               const hbfsim_kv_rotary_v1* rotary, void* stream);

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

/* Drafted tokens against the target's probabilities.  Sequence s has
 * d = counts[s] drafted tokens (clamped to [0, drafts]; NULL: drafts).  Token
 * i < d is accepted, as long as all before it are, if
 *   accept[i] * draft[i][token] < target[i][token]   (in 64 bits, exactly)
 * where `draft` NULL stands for 1 (tokens that were looked up, not drawn); a
 * token outside [0, vocab) is not.  With a accepted, the next token is drawn
 * from row a of the target: probabilities are read as whole multiples of
 * 2^-40, p40 = rint(p * 2^40) (halves to even; p clamped to [0, 1], NaN as 0),
 * with weights
 *   max(target40 - draft40, 0)   if a < d (draft NULL: target40, and 0 for the
 *                                token that was not accepted)
 *   target40                     if a = d, or if the former are all 0.
 * The next token is the least one whose inclusive sum of weights exceeds
 * floor(u * sum / 2^24), u = floor(sample * 2^24) within [0, 2^24) (NaN as 0);
 * -1 where every weight is 0.  Sums are whole numbers: results do not depend on
 * their order.
 * tokens_out: int32 [seqs][drafts + 1]: the accepted tokens, the next one, -1
 * behind.  accepted: int32 [seqs].  lengths_out (NULL to skip): lengths - (d -
 * a), the tokens that stay in the cache of a sequence whose `lengths` counts its
 * drafted ones.
 * Outputs lie in memory apart from the inputs' and from each other's, but
 * accepted may be counts' own memory and lengths_out that of lengths.
 * Limits: 32 drafts, 65536 sequences, a vocabulary of 2^22. */
enum hbfsim_kv_probability_type {
    HBFSIM_KV_P_BF16 = 0,
    HBFSIM_KV_P_F16 = 1,
    HBFSIM_KV_P_F32 = 2
};

typedef struct hbfsim_kv_verify_batch_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t type;               /* hbfsim_kv_probability_type of target and draft */
    uint32_t seqs;
    uint32_t drafts;
    uint32_t vocab;
    const void* target;          /* [seqs][drafts + 1][vocab], last axis contiguous */
    int64_t target_stride_seq;   /* in elements */
    int64_t target_stride_token;
    const void* draft;           /* [seqs][drafts][vocab] or NULL */
    int64_t draft_stride_seq;
    int64_t draft_stride_token;
    const int32_t* tokens;       /* [seqs][drafts] */
    const float* accept;         /* [seqs][drafts], in [0, 1) */
    const float* sample;         /* [seqs], in [0, 1) */
    const int32_t* counts;       /* [seqs] or NULL */
    const int32_t* lengths;      /* [seqs] or NULL */
    int32_t* accepted;
    int32_t* tokens_out;
    int32_t* lengths_out;
} hbfsim_kv_verify_batch_v1;

int hbfsim_kv_verify_v1(const hbfsim_kv_verify_batch_v1* batch, void* stream);

/* Pages.  refs (int32 [pages]) counts the table entries that name a page; a
 * page is free while its count is below 1.  Tables are as above, of blocks of
 * 16, 32 or 64 tokens; pages, seqs * width and the lists' entries are below
 * 2^31.  Outputs that have an input's type and shape (refs, table) may be that
 * input's own memory (for tables: with the same stride); everything else lies in
 * memory apart, where a table's memory is all from its lowest row to its highest.
 * Counts change by whole numbers: results do not depend on any order. */

/* Every sequence gets or gives back pages, so that it can hold want[s] tokens
 * of which it holds lengths[s] (both clamped to [0, width * block_tokens]).
 * In this order:
 *  - entries from block ceil(want / block_tokens) on become -1, and their pages'
 *    counts go down by one; so do the counts of listed pages (freed: int32
 *    [freed_rows][freed_width], the first freed_counts[...] of a row, as an
 *    eviction gives them; NULL: none).
 *  - if want > lengths, blocks from floor(lengths / block_tokens) on are asked
 *    for.  One without a page claims a free page; so does one whose page has a
 *    count above 1, unless the call asks for that page as often as it is
 *    counted and no later sequence does: then it stays.
 *  - claims are served in order of sequence and block by the free pages in
 *    ascending order.  The new page is counted once, a page that was left goes
 *    down by one.  Where the first asked block holds earlier tokens and left its
 *    page, src[s] and dst[s] say what to copy (hbfsim_kv_copy_v1, for every
 *    layer, before the append); else they are -1.
 * limits[s]: the tokens that sequence s may now be filled up to: want, or, where
 * free pages ran out, the beginning of its first block that was not served (a
 * page that stays is not served where one claim before it was not), but no less
 * than lengths.  Blocks that were not served stay as they were. */
typedef struct hbfsim_kv_resize_batch_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t seqs;
    uint32_t width;
    uint32_t block_tokens;
    uint32_t freed_rows;
    uint32_t freed_width;
    uint32_t reserved;
    uint64_t pages;
    const int32_t* refs;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* want;
    const int32_t* freed;
    const int32_t* freed_counts;
    int32_t* refs_out;
    int32_t* table_out;
    int64_t table_out_stride;
    int32_t* limits;
    int32_t* src;
    int32_t* dst;
    void* workspace;
    uint64_t workspace_bytes;
} hbfsim_kv_resize_batch_v1;

uint64_t hbfsim_kv_resize_workspace_v1(const hbfsim_kv_resize_batch_v1* batch);
int hbfsim_kv_resize_v1(const hbfsim_kv_resize_batch_v1* batch, void* stream);

/* Sequences go on as children of others: row r of the new table (int32
 * [rows][width]) is the row of parents[r], as far as its length reaches and -1
 * behind, or empty where parents[r] is outside [0, seqs).  Every entry of the old
 * table gives its page's count back, every entry of the new one takes one; a
 * block that is still filled is shared until hbfsim_kv_resize_v1 parts it.
 * lengths_out: int32 [rows].  table_out lies in memory apart from table. */
typedef struct hbfsim_kv_fork_batch_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t seqs;
    uint32_t rows;
    uint32_t width;
    uint32_t block_tokens;
    uint64_t pages;
    const int32_t* refs;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* parents;      /* [rows] */
    int32_t* refs_out;
    int32_t* table_out;          /* [rows][width] */
    int32_t* lengths_out;
} hbfsim_kv_fork_batch_v1;

int hbfsim_kv_fork_v1(const hbfsim_kv_fork_batch_v1* batch, void* stream);

/* Pages in use move to the front: with n of them, the highest at or past n goes
 * to the lowest free page, the next highest to the next.  src, dst (int32 [pages
 * / 2]): the moves in that order, -1 behind; live (int32 [1]): n; where (int32
 * [pages]): the place of every page in use, -1 for the others.  refs_out: the
 * counts at the new places, 0 from n on.  Entries of the table that name a page
 * become its new place (-1 for a free one); others stay. */
typedef struct hbfsim_kv_compact_batch_v1 {
    uint32_t struct_size;
    uint32_t version;
    uint32_t seqs;
    uint32_t width;
    uint64_t pages;
    const int32_t* refs;
    const int32_t* table;
    int64_t table_stride;
    int32_t* refs_out;
    int32_t* table_out;
    int64_t table_out_stride;
    int32_t* src;
    int32_t* dst;
    int32_t* live;
    int32_t* where;
    void* workspace;
    uint64_t workspace_bytes;
} hbfsim_kv_compact_batch_v1;

uint64_t hbfsim_kv_compact_workspace_v1(const hbfsim_kv_compact_batch_v1* batch);
int hbfsim_kv_compact_v1(const hbfsim_kv_compact_batch_v1* batch, void* stream);

/* Contents of pages: page dst[i] of `to` becomes page src[i] of `from` (data,
 * scale and bounds; the caches may be one) for i < count.  An entry outside its
 * pool, on either side, is passed over.  No page of dst may occur twice, nor
 * among the pages of src if the caches are one. */
int hbfsim_kv_copy_v1(const hbfsim_kv_cache_v1* from,
                      const hbfsim_kv_cache_v1* to, const int32_t* src,
                      const int32_t* dst, uint64_t count, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HBFSIM_KV_V1_H */
