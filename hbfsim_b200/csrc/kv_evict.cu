// kv_evict.cu -- blocks of least accumulated attention weight leave a block
// table (kv_v1.h).
//
// One CTA per sequence.  The weights become whole numbers (2^30 to a query)
// before anything is added, so scores and decisions do not depend on the
// order of the sums.  Pass 1 adds the step's weights to every block's score
// (kept in shared memory up to kHeldBlocks blocks, else in the output; few
// long sequences have it done by a kernel of its own over all SMs); the
// score of the last block to leave is found by a selection on the scores;
// the walk in block order then closes up the survivors.
#include "kv.h"

namespace hbfb {
namespace {

constexpr u32 kEvictThreads = 1024, kAddThreads = 128;
constexpr u32 kHeldBlocks = 24 * 1024;  // 192 KB of scores

struct EvictArgs {
    const i64* score;
    const float* weights;
    const int* table;
    i64 table_stride;
    const int* lengths;
    i64* score_out;
    int* table_out;
    int* lengths_out;
    int* freed;
    int* freed_counts;
    u32 heads, width, block, keep, sink, recent, decay;
};

// A signed score as an unsigned key of the same order.
__device__ __forceinline__ u64 score_key(i64 s) { return static_cast<u64>(s) ^ (u64{1} << 63); }

// The new score of block j.
__device__ __forceinline__ i64 new_score(const EvictArgs& a, u64 row, u32 j)
{
    const float* weights = a.weights + row * a.heads + j;
    i64 s = a.score[row + j];
    if (a.decay) s -= s >> a.decay;
#pragma unroll 8
    for (u32 h = 0; h < a.heads; ++h) {
        const float w = fminf(fmaxf(weights[static_cast<u64>(h) * a.width], 0.0f), 1048576.0f);
        s += __float2ll_rn(w * 1073741824.0f);
    }
    return s;
}

__global__ void __launch_bounds__(kAddThreads) add_kernel(const EvictArgs a)
{
    kv_let_next();
    const u32 seq = blockIdx.y, j = blockIdx.x * kAddThreads + threadIdx.x;
    const u32 blocks = (static_cast<u32>(kv_length(a.lengths, seq, a.width, a.block)) + a.block - 1) / a.block;
    const u64 row = static_cast<u64>(seq) * a.width;
    if (j < blocks) a.score_out[row + j] = new_score(a, row, j);
}

// `added`: add_kernel has put the new scores into score_out.
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictArgs a, bool added)
{
    kv_wait_before();
    extern __shared__ __align__(16) i64 held[];
    __shared__ KvSelectShared sm;
    const u32 seq = blockIdx.x;
    const int length = kv_length(a.lengths, seq, a.width, a.block);
    const u32 blocks = (static_cast<u32>(length) + a.block - 1) / a.block;
    const u32 leave = blocks > a.keep ? blocks - a.keep : 0;
    const u64 row = static_cast<u64>(seq) * a.width;
    const int* table = a.table + static_cast<i64>(seq) * a.table_stride;
    i64* score_out = a.score_out + row;
    i64* score = a.width <= kHeldBlocks && leave ? held : score_out;
    int* table_out = a.table_out + row;
    int* freed = a.freed + row;
    if (threadIdx.x == 0) {
        a.lengths_out[seq] = length - static_cast<int>(leave * a.block);
        a.freed_counts[seq] = static_cast<int>(leave);
    }
    const u32 from = a.sink, to = blocks - min(a.recent, blocks);  // those that may leave
    u64 least = ~u64{0}, greatest = 0;
    // pass 1: every block's new score
    for (u32 j = threadIdx.x; j < a.width; j += blockDim.x) {
        if (j < blocks) {
            const i64 s = added ? score_out[j] : new_score(a, row, j);
            score[j] = s;
            if (leave == 0) table_out[j] = table[j];
            if (j >= from && j < to) {
                least = min(least, score_key(s));
                greatest = max(greatest, score_key(s));
            }
        }
        if (j >= blocks - leave) {  // behind the survivors
            if (j >= blocks || score != score_out) score_out[j] = 0;
            table_out[j] = -1;
        }
        if (j >= leave) freed[j] = -1;
    }
    if (leave == 0) return;
    __syncthreads();
    // the score of the last block to leave, and how many of its equals do
    u64 limit;
    u32 equals;
    kv_rank_limit<u64>(
        to, leave, least, greatest,
        [&](u32 j, u64& k) {
            k = score_key(score[j]);
            return j >= from;
        },
        sm, limit, equals);
    struct Entry {
        i64 score;
        int page;
    };
    auto state = [&](u32 j) -> u32 {
        if (j < from || j >= to) return 0;
        const u64 k = score_key(score[j]);
        return k < limit ? 1 : k == limit ? 2 : 0;
    };
    auto load = [&](u32 j) { return Entry{score[j], table[j]}; };
    auto store = [&](u32 j, const Entry& e, bool gone, u32 gone_before) {
        if (gone) {
            freed[gone_before] = e.page;
        } else {  // survivors only move towards the front
            score_out[j - gone_before] = e.score;
            table_out[j - gone_before] = e.page;
        }
    };
    if (score != score_out) kv_walk<false>(blocks, equals, sm, state, load, store);
    else kv_walk<true>(blocks, equals, sm, state, load, store);
    if (score == score_out) {  // what lies behind the survivors was needed until now
        __syncthreads();
        for (u32 j = blocks - leave + threadIdx.x; j < blocks; j += blockDim.x) score_out[j] = 0;
    }
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" int hbfsim_kv_evict_v1(const hbfsim_kv_evict_batch_v1* b, void* stream)
{
    if (!b || b->struct_size != sizeof(*b) || b->version != HBFSIM_KV_V1_VERSION)
        return HBFSIM_INVALID_ARGUMENT;
    if (b->block_tokens != 16 && b->block_tokens != 32 && b->block_tokens != 64)
        return HBFSIM_UNSUPPORTED;
    if (b->seqs > kKvMaxSeqs || b->width > kKvMaxWidth || b->kv_heads == 0 ||
        b->kv_heads > kKvMaxHeads || b->decay > 63 || b->recent == 0 ||
        static_cast<u64>(b->sink) + b->recent > b->keep ||
        static_cast<u64>(b->width) * b->block_tokens > 0x7fffffffull)
        return HBFSIM_INVALID_ARGUMENT;
    if (b->seqs == 0) return HBFSIM_OK;
    if (!b->lengths || !b->lengths_out || !b->freed_counts ||
        (b->width && (!b->score || !b->weights || !b->table || !b->score_out || !b->table_out ||
                      !b->freed)))
        return HBFSIM_INVALID_ARGUMENT;
    if (b->width && (b->score == b->score_out || b->table == b->table_out))
        return HBFSIM_INVALID_ARGUMENT;
    if (!kv_aligned(b->score, 8) || !kv_aligned(b->score_out, 8) || !kv_aligned(b->weights, 4) ||
        !kv_aligned(b->table, 4) || !kv_aligned(b->table_out, 4) || !kv_aligned(b->freed, 4))
        return HBFSIM_INVALID_ARGUMENT;
    EvictArgs a{b->score,      b->weights, b->table,        b->table_stride, b->lengths,
                b->score_out,  b->table_out, b->lengths_out, b->freed,       b->freed_counts,
                b->kv_heads,   b->width,   b->block_tokens, b->keep,         b->sink,
                b->recent,     b->decay};
    static std::atomic<u64> seen{0};
    if (!kv_allow_smem(evict_kernel, kHeldBlocks * 8, seen)) return HBFSIM_CUDA_ERROR;
    const u32 smem = b->width <= kHeldBlocks ? b->width * 8 : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Fewer sequences than half the SMs and more than two rounds of a CTA each: all SMs add.
    const bool apart = b->seqs * 2 < static_cast<u32>(kv_sm_count()) && b->width > 2 * kEvictThreads;
    if (apart)
        add_kernel<<<dim3((b->width + kAddThreads - 1) / kAddThreads, b->seqs), kAddThreads, 0, s>>>(a);
    const bool ok = kv_launch_behind(evict_kernel, dim3(b->seqs), kEvictThreads, s, smem, a, apart);
    return cudaGetLastError() == cudaSuccess && ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
