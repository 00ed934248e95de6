// kv_evict.cu -- blocks of least accumulated attention weight leave a block
// table (kv_v1.h).
//
// One team (a CTA, or a cluster with few long sequences) per sequence.  The
// weights become whole numbers (2^30 to a query) before anything is added, so
// scores and decisions do not depend on the order of the sums.  Pass 1 adds
// the step's weights to every block's score (kept in shared memory up to
// kHeldBlocks blocks a CTA, else in the output); the score of the last block
// to leave is found by a selection on the scores; the walk in block order
// then closes up the survivors.
//
// 64 tables of up to 2048 blocks with 8 heads take 10 us (5 MB), one of 16385
// blocks 13 us with a team of 8: a chain of a dozen barriers, not memory.
#include "kv.h"

#include <algorithm>

namespace hbfb {
namespace {

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

// `slice`: blocks of a row that one CTA of the team has.
__global__ void __launch_bounds__(1024) evict_kernel(const EvictArgs a, u32 team_size, u32 slice)
{
    extern __shared__ __align__(16) i64 held[];
    __shared__ KvSelectShared sm;
    const KvTeam team{blockIdx.x % team_size, team_size};
    const u32 seq = blockIdx.x / team_size;
    const int length = kv_length(a.lengths, seq, a.width, a.block);
    const u32 blocks = (static_cast<u32>(length) + a.block - 1) / a.block;
    const u32 leave = blocks > a.keep ? blocks - a.keep : 0;
    const u64 row = static_cast<u64>(seq) * a.width;
    const u32 first = team.rank * slice, end = min(first + slice, a.width);  // this CTA's
    const int* table = a.table + static_cast<i64>(seq) * a.table_stride;
    i64* score_out = a.score_out + row;
    const bool hold = slice <= kHeldBlocks && leave;
    i64* score = hold ? held : score_out + first;  // of block `first` on
    int* table_out = a.table_out + row;
    int* freed = a.freed + row;
    if (threadIdx.x == 0 && team.rank == 0) {
        a.lengths_out[seq] = length - static_cast<int>(leave * a.block);
        a.freed_counts[seq] = static_cast<int>(leave);
    }
    const u32 from = a.sink, to = blocks - min(a.recent, blocks);  // those that may leave
    u64 least = ~u64{0}, greatest = 0;
    // pass 1: every block's new score
    for (u32 j = first + threadIdx.x; j < end; j += blockDim.x) {
        if (j < blocks) {
            const i64 s = new_score(a, row, j);
            score[j - first] = s;
            if (leave == 0) table_out[j] = table[j];
            if (j >= from && j < to) {
                least = min(least, score_key(s));
                greatest = max(greatest, score_key(s));
            }
        }
        if (j >= blocks - leave) {  // behind the survivors
            if (j >= blocks || hold) score_out[j] = 0;
            table_out[j] = -1;
        }
        if (j >= leave) freed[j] = -1;
    }
    if (leave == 0) return;
    u32 none0 = 0, none1 = 0;
    kv_gather(team, sm, least, greatest, none0, none1);
    // the score of the last block to leave, and how many of its equals do
    u64 limit;
    u32 equals;
    const u32 mine = min(max(blocks, first), end) - first;  // blocks of this CTA in use
    kv_rank_limit<u64>(
        team, mine, leave, least, greatest,
        [&](u32 i, u64& k) {
            k = score_key(score[i]);
            return first + i >= from && first + i < to;
        },
        sm, limit, equals);
    struct Entry {
        i64 score;
        int page;
    };
    auto state = [&](u32 i) -> u32 {
        if (first + i < from || first + i >= to) return 0;
        const u64 k = score_key(score[i]);
        return k < limit ? 1 : k == limit ? 2 : 0;
    };
    auto load = [&](u32 i) { return i < mine ? Entry{score[i], table[first + i]} : Entry{0, 0}; };
    auto store = [&](u32 i, const Entry& e, bool gone, u32 gone_before) {
        if (gone) {
            freed[gone_before] = e.page;
        } else {  // survivors only move towards the front
            score_out[first + i - gone_before] = e.score;
            table_out[first + i - gone_before] = e.page;
        }
    };
    if (hold) kv_walk<false, false>(team, mine, equals, sm, state, load, store);
    else kv_walk<true, false>(team, mine, equals, sm, state, load, store);
    kv_team_sync(team);  // nobody leaves while another may read its counts
    if (!hold)  // what lies behind the survivors was needed until now
        for (u32 j = blocks - leave + threadIdx.x; j < blocks; j += blockDim.x) score_out[j] = 0;
}

struct Memory {
    std::uintptr_t from, end;
    Memory(const void* p, u64 bytes) : from(reinterpret_cast<std::uintptr_t>(p)), end(from + bytes) {}
    bool meets(const Memory& other) const { return from < other.end && other.from < end; }
};

// Whether an output lies in an input's memory or in another output's: every thread block writes its
// outputs while others still read.
bool would_race(const hbfsim_kv_evict_batch_v1& b)
{
    const u64 seqs = b.seqs, row = u64{b.width} * 4;
    const Memory out[] = {{b.score_out, seqs * row * 2}, {b.table_out, seqs * row}, {b.lengths_out, seqs * 4},
                          {b.freed, seqs * row}, {b.freed_counts, seqs * 4}};
    const Memory in[] = {{b.score, seqs * row * 2}, {b.weights, seqs * b.kv_heads * row}, {b.lengths, seqs * 4}};
    // the table's rows, from the first to the last; one by one only where something lies among them
    const int* last = b.table + static_cast<i64>(seqs - 1) * b.table_stride;
    const Memory table(std::min(b.table, last), reinterpret_cast<std::uintptr_t>(std::max(b.table, last)) -
                                                    reinterpret_cast<std::uintptr_t>(std::min(b.table, last)) + row);
    for (const Memory& o : out) {
        for (const Memory& i : in)
            if (o.meets(i)) return true;
        for (const Memory* p = out; p != &o; ++p)
            if (o.meets(*p)) return true;
        if (o.meets(table))
            for (u64 s = 0; s < seqs; ++s)
                if (o.meets(Memory(b.table + static_cast<i64>(s) * b.table_stride, row))) return true;
    }
    return false;
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
    if (!kv_aligned(b->score, 8) || !kv_aligned(b->score_out, 8) || !kv_aligned(b->weights, 4) ||
        !kv_aligned(b->table, 4) || !kv_aligned(b->table_out, 4) || !kv_aligned(b->freed, 4) ||
        !kv_aligned(b->lengths, 4) || !kv_aligned(b->lengths_out, 4) || !kv_aligned(b->freed_counts, 4))
        return HBFSIM_INVALID_ARGUMENT;
    if (would_race(*b)) return HBFSIM_INVALID_ARGUMENT;
    EvictArgs a{b->score,      b->weights, b->table,        b->table_stride, b->lengths,
                b->score_out,  b->table_out, b->lengths_out, b->freed,       b->freed_counts,
                b->kv_heads,   b->width,   b->block_tokens, b->keep,         b->sink,
                b->recent,     b->decay};
    static std::atomic<u64> seen{0};
    if (!kv_allow_smem(evict_kernel, kHeldBlocks * 8, seen)) return HBFSIM_CUDA_ERROR;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    u32 team = kv_team_size(b->seqs, b->width);
    u32 slice = (b->width + team - 1) / team;
    if (slice > kHeldBlocks) {  // a row that no team can hold is walked in place by one CTA
        team = 1;
        slice = b->width;
    }
    const bool ok = kv_launch(evict_kernel, dim3(b->seqs * team), kv_team_threads(slice), s,
                              slice <= kHeldBlocks ? slice * 8 : 0, team, false, a, team, slice);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
