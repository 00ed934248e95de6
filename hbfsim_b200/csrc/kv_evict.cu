// kv_evict.cu -- blocks of least accumulated attention weight leave a block
// table (kv_v1.h).
//
// One CTA per sequence.  The weights become whole numbers (2^30 to a query)
// before anything is added, so scores and decisions do not depend on the
// order of the sums.  Pass 1 adds the step's weights to every block's score;
// the score of the last block to leave is found by a radix selection on the
// scores; pass 2 walks the blocks in order and closes up the survivors with
// block-wide scans.
#include "kv.h"

namespace hbfb {
namespace {

constexpr u32 kEvictThreads = 1024;

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

__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictArgs a)
{
    __shared__ u32 histogram[256];
    __shared__ u32 shared2[2];
    __shared__ u32 warp_sums[33];
    const u32 seq = blockIdx.x;
    const int length = kv_length(a.lengths, seq, a.width, a.block);
    const u32 blocks = (static_cast<u32>(length) + a.block - 1) / a.block;
    const u32 leave = blocks > a.keep ? blocks - a.keep : 0;
    const u64 row = static_cast<u64>(seq) * a.width;
    const i64* score_in = a.score + row;
    const float* weights = a.weights + row * a.heads;
    const int* table = a.table + static_cast<i64>(seq) * a.table_stride;
    i64* score = a.score_out + row;
    int* table_out = a.table_out + row;
    int* freed = a.freed + row;
    if (threadIdx.x == 0) {
        a.lengths_out[seq] = length - static_cast<int>(leave * a.block);
        a.freed_counts[seq] = static_cast<int>(leave);
    }
    // pass 1: every block's new score, at its old place
    for (u32 j = threadIdx.x; j < a.width; j += blockDim.x) {
        i64 s = 0;
        if (j < blocks) {
            s = score_in[j];
            if (a.decay) s -= s >> a.decay;
            for (u32 h = 0; h < a.heads; ++h) {
                const float w = fminf(fmaxf(weights[static_cast<u64>(h) * a.width + j], 0.0f), 1048576.0f);
                s += __float2ll_rn(w * 1073741824.0f);
            }
        }
        score[j] = s;
        freed[j] = -1;
        if (leave == 0) table_out[j] = j < blocks ? table[j] : -1;
    }
    if (leave == 0) return;
    __syncthreads();
    // the score of the last block to leave, and how many of its equals do
    const u32 from = a.sink, to = blocks - a.recent;
    u32 below;
    const u64 limit = kv_select_rank<u64>(
        blocks, leave,
        [&](u32 j, u64& k) {
            k = score_key(score[j]);
            return j >= from && j < to;
        },
        histogram, shared2, below);
    const u32 equals = leave - below;
    // pass 2: tiles of blocks in order; a tile is read before it is written,
    // and survivors only move towards the front
    u32 gone_before = 0, equal_before = 0;
    for (u32 base = 0; base < blocks; base += blockDim.x) {
        const u32 j = base + threadIdx.x;
        i64 s = 0;
        int page = -1;
        u64 key = ~u64{0};
        const bool in = j < blocks;
        if (in) {
            s = score[j];
            page = table[j];
            key = score_key(s);
        }
        const bool may = in && j >= from && j < to;
        const u32 equal = may && key == limit ? 1u : 0u;
        const u32 equal_upto = equal_before + kv_block_scan(equal, warp_sums);
        equal_before += warp_sums[32];
        const u32 gone = may && (key < limit || (equal && equal_upto <= equals)) ? 1u : 0u;
        const u32 gone_upto = gone_before + kv_block_scan(gone, warp_sums);
        gone_before += warp_sums[32];
        if (gone) freed[gone_upto - 1] = page;
        else if (in) {
            score[j - gone_upto] = s;
            table_out[j - gone_upto] = page;
        }
    }
    __syncthreads();
    for (u32 j = blocks - leave + threadIdx.x; j < a.width; j += blockDim.x) {
        score[j] = 0;
        table_out[j] = -1;
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
    evict_kernel<<<b->seqs, kEvictThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return cudaGetLastError() == cudaSuccess ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
