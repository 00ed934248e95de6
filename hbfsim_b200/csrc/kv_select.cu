// kv_select.cu -- block lists by a cheap score (kv_v1.h).
//
// A group's score of a block is linear in the block's bounds once the
// queries are split by sign: sum_d up_d * hi_d + down_d * lo_d with
// up = sum_g max(qi, 0), down = sum_g min(qi, 0).  So a block costs one dot
// product of 2 * head_dim channels per group instead of one per query head,
// and 2 * head_dim bytes, 1/16 of its keys and values at 16 tokens a block.
// The sums go through the tensor cores as 8-bit whole numbers: up and down
// (at most 64 * 127) are split into 128 * high + low, two columns of the
// narrow side; 16 blocks of a head are the wide side, read straight into the
// fragments, 16 bytes per lane.  (Two-way dot instructions took 4 times the
// instructions and were bound by them.)
//
// score_kernel streams the bounds and writes a 32-bit ordered key per
// (token, head, block): the blocks of all sequences form one line that is cut
// into equal shares, one per resident CTA.  list_kernel, one team (a CTA, or
// a cluster for few long rows) per (sequence, token, head), finds the key of
// the last block to list by a selection on the keys (in shared memory up to
// kHeldKeys blocks a CTA) and writes the list in block order.
#include "kv.h"

#include <algorithm>

namespace hbfb {
namespace {

constexpr u32 kScoreThreads = 256, kScorePerSm = 3;
constexpr u32 kScoreShare = 32;      // blocks of a CTA at least
constexpr u32 kHeldKeys = 32 * 1024; // 128 KB of keys
constexpr u32 kMostQueryBytes = 200 * 1024;  // of shared memory, for the whole-number queries
constexpr u32 kAbsent = 0u;           // key of a block that cannot be listed
constexpr u32 kAlways = 0xffffffffu;  // key of a block that is always listed

struct SelectArgs {
    KvView c;
    KvQuery q;
    u32 top, sink, recent;
    u32* keys;  // [seqs][tokens][heads][width]
    int* blocks;
    int* counts;
};

// E neighbouring channels of a query, those that are not finite as 0.
template <int E>
__device__ __forceinline__ void query_at(const KvQuery& q, u32 seq, u32 token, u32 head, u32 d,
                                         float (&x)[E])
{
    const i64 at = static_cast<i64>(seq) * q.stride_seq + static_cast<i64>(token) * q.stride_token +
                   static_cast<i64>(head) * q.stride_head + d;
    kv_load<E>(q.q, at, q.type, q.wide, x);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fabsf(x[e]) <= 3.402823466e38f ? x[e] : 0.0f;
}

// Blocks that a query token may look at: those up to its own position.
__device__ __forceinline__ u32 blocks_of_token(int length, u32 tokens, u32 t, u32 block)
{
    const int last = length - static_cast<int>(tokens) + static_cast<int>(t);
    return last < 0 ? 0u : (static_cast<u32>(last) >> (31 - __clz(block))) + 1u;  // 16, 32 or 64
}

// Finite floats in their order, above kAbsent and below kAlways.
__device__ __forceinline__ u32 order_key(float x)
{
    const u32 b = __float_as_uint(fminf(x, 3.402823466e38f) + 0.0f);  // -0 becomes 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ u32 blocks_of_sequence(const SelectArgs& a, u32 seq)
{
    return blocks_of_token(kv_length(a.q.lengths, seq, a.q.width, a.c.block), a.q.tokens,
                           a.q.tokens - 1, a.c.block);
}

// Bytes between the columns (token, high or low) of a head's whole-number
// queries in shared memory: down then up, and padding that puts neighbouring
// columns on different banks.
HD constexpr u32 column_bytes(u32 dim) { return 2 * dim + 64; }

__device__ __forceinline__ void mma16832(int (&d)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int D>
__global__ void __launch_bounds__(kScoreThreads, kScorePerSm) score_kernel(const SelectArgs a)
{
    constexpr u32 kChunks = D / 32;  // 16-byte pieces of a block's bounds per lane
    constexpr u32 kColumn = column_bytes(D);
    extern __shared__ __align__(16) std::int8_t whole[];  // [heads][2 tokens][kColumn]
    __shared__ u64 line;
    kv_let_next();
    const u32 heads = a.c.heads, tokens = a.q.tokens, group = a.q.group;
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = kScoreThreads / 32;
    // the line of all sequences' blocks, and this CTA's share of it
    u64 all = 0;
    for (u32 s = threadIdx.x; s < a.q.seqs; s += kScoreThreads) all += blocks_of_sequence(a, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (threadIdx.x == 0) line = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&line), all);
    __syncthreads();
    const u64 share = max(static_cast<u64>(kScoreShare), (line + gridDim.x - 1) / gridDim.x);
    u64 at = blockIdx.x * share;
    const u64 stop = min(at + share, line);
    if (at >= stop) return;
    u32 seq = 0, have = 0;
    u64 begin = 0;
    for (u32 base = 0; base < a.q.seqs; base += 32) {  // the sequence that holds `at`
        const u32 n = base + lane < a.q.seqs ? blocks_of_sequence(a, base + lane) : 0;
        u32 upto = n;
#pragma unroll
        for (u32 o = 1; o < 32; o <<= 1) {
            const u32 y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const u32 holds = __ballot_sync(0xffffffffu, at < begin + upto);
        if (holds) {
            const int k = __ffs(holds) - 1;
            seq = base + k;
            have = __shfl_sync(0xffffffffu, n, k);
            begin += __shfl_sync(0xffffffffu, upto - n, k);
            break;
        }
        begin += __shfl_sync(0xffffffffu, upto, 31);
    }
    for (; at < stop; begin += have, have = ++seq < a.q.seqs ? blocks_of_sequence(a, seq) : 0) {
        const u32 first = static_cast<u32>(at - begin);
        const u32 end = static_cast<u32>(min(stop - begin, static_cast<u64>(have)));
        if (first >= end) continue;
        at = begin + end;
        const int length = kv_length(a.q.lengths, seq, a.q.width, a.c.block);
        __syncthreads();  // the queries of the sequence before are used
        for (u32 th = warp; th < tokens * heads; th += warps) {
            const u32 t = th / heads, h = th % heads;
            constexpr int E = D / 32;  // channels of a lane
            float most = 0.0f;
#pragma unroll 4
            for (u32 i = 0; i < group; ++i) {
                float x[E];
                query_at<E>(a.q, seq, t, h * group + i, lane * E, x);
#pragma unroll
                for (int e = 0; e < E; ++e) most = fmaxf(most, fabsf(x[e]));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            int x = 0;
            frexpf(most, &x);
            const float up_scale = kv_power(7 - max(x, -100));
            int up[E], down[E];
#pragma unroll
            for (int e = 0; e < E; ++e) up[e] = down[e] = 0;
#pragma unroll 4
            for (u32 i = 0; i < group; ++i) {
                float x[E];
                query_at<E>(a.q, seq, t, h * group + i, lane * E, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float r = rintf(x[e] * up_scale);
                    const int qi = static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
                    up[e] += max(qi, 0);
                    down[e] += min(qi, 0);
                }
            }
            // column 2 t: the high parts, 2 t + 1: the low ones; first down, then up
            std::int8_t* to = whole + (h * 2 * tokens + 2 * t) * kColumn + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                to[e] = static_cast<std::int8_t>(-(-down[e] >> 7));
                to[kColumn + e] = static_cast<std::int8_t>(-(-down[e] & 127));
                to[D + e] = static_cast<std::int8_t>(up[e] >> 7);
                to[D + kColumn + e] = static_cast<std::int8_t>(up[e] & 127);
            }
        }
        __syncthreads();
        const int* table = a.q.table + static_cast<i64>(seq) * a.q.table_stride;
        const u32 g = lane >> 2, c = lane & 3u;
        // Tasks: 16 blocks of one head, heads first, by the warps in turn.
        const u32 rows = (end - first + 15) / 16, skip_rows = warps / heads, skip_heads = warps % heads;
        auto page_of = [&](u32 row, u32 more) {
            const u32 j = first + row * 16 + g + more;
            return row < rows && j < end ? kv_page(table, j, a.c.pages) : -1;
        };
        u32 row = warp / heads, h = warp % heads;
        int next0 = page_of(row, 0), next1 = page_of(row, 8);
        while (row < rows) {
            const u32 j0 = first + row * 16 + g, j1 = j0 + 8, head = h;
            const int page0 = next0, page1 = next1;
            row += skip_rows;
            h += skip_heads;
            if (h >= heads) {
                h -= heads;
                ++row;
            }
            uint4 x0[kChunks], x1[kChunks];
            float scale0 = 0.0f, scale1 = 0.0f;
#pragma unroll
            for (u32 k = 0; k < kChunks; ++k) x0[k] = x1[k] = make_uint4(0, 0, 0, 0);
            if (page0 >= 0) {
                const u64 x = static_cast<u64>(page0) * heads + head;
                const uint4* b = reinterpret_cast<const uint4*>(a.c.bounds + x * 2 * D) + c;
#pragma unroll
                for (u32 k = 0; k < kChunks; ++k) x0[k] = b[k * 4];
                scale0 = a.c.scale[x * 2];
            }
            if (page1 >= 0) {
                const u64 x = static_cast<u64>(page1) * heads + head;
                const uint4* b = reinterpret_cast<const uint4*>(a.c.bounds + x * 2 * D) + c;
#pragma unroll
                for (u32 k = 0; k < kChunks; ++k) x1[k] = b[k * 4];
                scale1 = a.c.scale[x * 2];
            }
            next0 = page_of(row, 0);
            next1 = page_of(row, 8);
            // four tokens at a time: column g is the high or low part of token t0 + g / 2
            for (u32 t0 = 0; t0 < tokens; t0 += 4) {
                int s0[4] = {0, 0, 0, 0}, s1[4] = {0, 0, 0, 0};
                const bool used = t0 + g / 2 < tokens;
                const std::int8_t* column = whole + (head * 2 * tokens + 2 * t0 + g) * kColumn + c * 16;
#pragma unroll
                for (u32 k = 0; k < kChunks; ++k) {
                    uint4 y = make_uint4(0, 0, 0, 0);
                    if (used) y = *reinterpret_cast<const uint4*>(column + k * 64);
                    mma16832(s0, x0[k].x, x1[k].x, x0[k].y, x1[k].y, y.x, y.y);
                    mma16832(s1, x0[k].z, x1[k].z, x0[k].w, x1[k].w, y.z, y.w);
                }
                const u32 t = t0 + c;  // this lane's columns 2c and 2c + 1
                if (t < tokens) {
                    const u32 mine = blocks_of_token(length, tokens, t, a.c.block);
                    u32* keys = a.keys + ((static_cast<u64>(seq) * tokens + t) * heads + head) * a.q.width;
                    auto put = [&](u32 j, int page, int sum, float scale) {
                        u32 key = kAbsent;
                        if (page >= 0 && j < mine)
                            key = j < a.sink || j + a.recent >= mine
                                      ? kAlways
                                      : order_key(__fmul_rn(__int2float_rn(sum), scale));
                        if (j < end) keys[j] = key;
                    };
                    put(j0, page0, (s0[0] + s1[0]) * 128 + s0[1] + s1[1], scale0);
                    put(j1, page1, (s0[2] + s1[2]) * 128 + s0[3] + s1[3], scale1);
                }
            }
        }
    }
}

// `slice`: blocks of a row that one CTA of the team has.
__global__ void __launch_bounds__(1024) list_kernel(const SelectArgs a, u32 team_size, u32 slice)
{
    extern __shared__ __align__(16) u32 held[];
    __shared__ KvSelectShared sm;
    __shared__ u32 counted[4];  // blocks that are there, those always listed; the team's
    kv_wait_before();
    const KvTeam team{blockIdx.x % team_size, team_size};
    const u64 at = blockIdx.x / team_size;  // (sequence, token, head)
    const u32 heads = a.c.heads, tokens = a.q.tokens;
    const u32 t = static_cast<u32>(at / heads % tokens), seq = static_cast<u32>(at / heads / tokens);
    const int length = kv_length(a.q.lengths, seq, a.q.width, a.c.block);
    const u32 have = blocks_of_token(length, tokens, t, a.c.block);
    const u32 first = team.rank * slice, mine = min(max(have, first), first + slice) - first;
    const u32* row = a.keys + at * a.q.width + first;
    const bool hold = slice <= kHeldKeys;
    const u32* keys = hold ? held : row;
    int* list = a.blocks + at * a.top;
    if (threadIdx.x < 2) counted[threadIdx.x] = 0;
    __syncthreads();
    u32 there = 0, always = 0, least = ~0u, greatest = 0;
#pragma unroll 8
    for (u32 i = threadIdx.x; i < mine; i += blockDim.x) {
        const u32 k = row[i];
        if (hold) held[i] = k;
        there += k != kAbsent;
        always += k == kAlways;
        if (k != kAbsent && k != kAlways) {
            least = min(least, ~k);
            greatest = max(greatest, ~k);
        }
    }
    there = __reduce_add_sync(0xffffffffu, there);
    always = __reduce_add_sync(0xffffffffu, always);
    if ((threadIdx.x & 31u) == 0) {
        atomicAdd(&counted[0], there);
        atomicAdd(&counted[1], always);
    }
    kv_team_sync(team);
    if (team.size > 1) {
        if (threadIdx.x < 32) {
            const u32 all = kv_team_sum(&counted[0], team.size), all_always = kv_team_sum(&counted[1], team.size);
            if (threadIdx.x == 0) {
                counted[2] = all;
                counted[3] = all_always;
            }
        }
        __syncthreads();
    }
    there = counted[team.size > 1 ? 2 : 0];
    always = counted[team.size > 1 ? 3 : 1];
    const u32 take = min(a.top, there);
    // the greatest keys are the smallest of their complements; those always listed need no rank
    u32 limit = 0xffffffffu, equals = kKvAll;
    if (take < there && take > always)
        kv_rank_limit<u32>(
            team, mine, take - always, least, greatest,
            [&](u32 i, u32& k) {
                k = keys[i];
                if (k == kAbsent || k == kAlways) return false;
                k = ~k;
                return true;
            },
            sm, limit, equals);
    else if (take < there)
        limit = 0, equals = 0;  // none but those always listed
    kv_walk<false>(
        team, mine, equals, sm,
        [&](u32 i) -> u32 {
            const u32 k = keys[i];
            if (k == kAbsent) return 0;
            return k == kAlways || ~k < limit ? 1 : ~k == limit ? 2 : 0;
        },
        [](u32) { return 0; },
        [&](u32 i, int, bool listed, u32 before) {
            if (listed && before < a.top) list[before] = static_cast<int>(first + i);
        });
    if (team.rank == 0) {
        for (u32 i = take + threadIdx.x; i < a.top; i += blockDim.x) list[i] = -1;
        if (threadIdx.x == 0) a.counts[at] = static_cast<int>(take);
    }
    kv_team_sync(team);  // nobody leaves while another may read its counts
}

u64 workspace_bytes_of(const KvView& v, const KvQuery& q)
{
    return kv_round_up(static_cast<u64>(q.seqs) * q.tokens * v.heads * q.width * 4, 256);
}

template <int D>
int launch(const SelectArgs& a, cudaStream_t s)
{
    const u32 smem = a.q.tokens * a.c.heads * 2 * column_bytes(D);
    static std::atomic<u64> seen{0};
    if (!kv_allow_smem(score_kernel<D>, kMostQueryBytes, seen)) return HBFSIM_CUDA_ERROR;
    const u64 most = (static_cast<u64>(a.q.seqs) * a.q.width + kScoreShare - 1) / kScoreShare;
    const u32 grid = static_cast<u32>(std::min<u64>(most, static_cast<u64>(kScorePerSm) * kv_sm_count()));
    if (grid) score_kernel<D><<<grid, kScoreThreads, smem, s>>>(a);
    static std::atomic<u64> seen_list{0};
    if (!kv_allow_smem(list_kernel, kHeldKeys * 4, seen_list)) return HBFSIM_CUDA_ERROR;
    const u32 rows = a.q.seqs * a.q.tokens * a.c.heads;
    u32 team = kv_team_size(rows, a.q.width), slice = (a.q.width + team - 1) / team;
    if (slice > kHeldKeys) {  // a row that no team can hold is one CTA's
        team = 1;
        slice = a.q.width;
    }
    // many rows: small CTAs, several to an SM
    u32 threads = kv_team_threads(slice);
    if (rows > 2 * static_cast<u32>(kv_sm_count())) threads = std::min(threads, 256u);
    const bool ok = kv_launch_behind(list_kernel, dim3(rows * team), threads, s,
                                     slice <= kHeldKeys ? slice * 4 : 0, team, a, team, slice);
    return cudaGetLastError() == cudaSuccess && ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" uint64_t hbfsim_kv_select_workspace_v1(const hbfsim_kv_cache_v1* cache,
                                                  const hbfsim_kv_query_v1* query)
{
    KvView v{};
    KvQuery q{};
    if (kv_check_cache(cache, v) || kv_check_query(query, v, q)) return 0;
    return workspace_bytes_of(v, q);
}

extern "C" int hbfsim_kv_select_v1(const hbfsim_kv_cache_v1* cache,
                                   const hbfsim_kv_query_v1* query, uint32_t top, uint32_t sink,
                                   uint32_t recent, int32_t* blocks, int32_t* counts,
                                   void* workspace, uint64_t workspace_bytes, void* stream)
{
    SelectArgs a{};
    if (const int rc = kv_check_cache(cache, a.c)) return rc;
    if (const int rc = kv_check_query(query, a.c, a.q)) return rc;
    if (top == 0 || top > kKvMaxWidth || recent == 0 ||
        static_cast<u64>(sink) + recent > top)
        return HBFSIM_INVALID_ARGUMENT;
    const u64 lists = static_cast<u64>(a.q.seqs) * a.q.tokens * a.c.heads;
    if (lists == 0) return HBFSIM_OK;
    // shared memory of the whole-number queries
    if (static_cast<u64>(a.q.tokens) * a.c.heads * 2 * column_bytes(a.c.dim) > kMostQueryBytes)
        return HBFSIM_UNSUPPORTED;
    if (!blocks || !counts) return HBFSIM_INVALID_ARGUMENT;
    if (workspace_bytes < workspace_bytes_of(a.c, a.q) || (a.q.width && !workspace) ||
        !kv_aligned(workspace, 16) || !kv_aligned(blocks, 4) || !kv_aligned(counts, 4))
        return HBFSIM_INVALID_ARGUMENT;
    a.top = top;
    a.sink = sink;
    a.recent = recent;
    a.keys = static_cast<u32*>(workspace);
    a.blocks = blocks;
    a.counts = counts;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.c.dim == 64) return launch<64>(a, s);
    if (a.c.dim == 128) return launch<128>(a, s);
    return launch<256>(a, s);
}
