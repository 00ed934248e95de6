// kv_select.cu -- block lists by a cheap score (kv_v1.h).
//
// A group's score of a block is linear in the block's bounds once the
// queries are split by sign: sum_d up_d * hi_d + down_d * lo_d with
// up = sum_g max(qi, 0), down = sum_g min(qi, 0).  So a block costs one dot
// product of 2 * head_dim channels per group instead of one per query head,
// and 2 * head_dim bytes, 1/16 of its keys and values at 16 tokens a block.
// The sums go through the tensor cores as 8-bit whole numbers: up and down
// (at most 64 * 127) are split into 128 * high + low, two columns of the
// narrow side; 16 blocks of a head are the wide side.  (Two-way dot
// instructions took 4 times the instructions and were bound by them.)
//
// query_kernel makes the whole numbers once; score_kernel streams the bounds
// through a ring of asynchronous copies per warp and writes a 32-bit ordered
// key per (token, head, block): the blocks of all sequences form one line
// that is cut into equal shares, one per resident CTA.  Then the key of the
// last block to list is found for every (sequence, token, head), and the list
// is written in block order: by short_list_kernel, a CTA per row with the keys
// in registers, up to kShortRow blocks; else by list_kernel, a team (a CTA, or
// a cluster for few long rows) per row with the keys in shared memory up to
// kHeldKeys a CTA.  Each kernel is set up while the one before it runs.
//
// One decode step of 64 sequences of 1024 to 32768 tokens, 8 heads of 128
// channels, blocks of 16: 41 us.  score_kernel takes 31 us of them, 143 MB of
// bounds in pieces of 256 bytes at 4.6 TB/s (71 % of a copy's rate, 41 % of
// the issue slots), short_list_kernel 8 us, a barrier for each of some 20 bits.
#include "kv.h"

#include <algorithm>

namespace hbfb {
namespace {

constexpr u32 kQueryWarps = 4;
constexpr u32 kScoreWarps = 8;
constexpr u32 kScoreShare = 32;      // blocks of a CTA at least
constexpr u32 kHeldKeys = 32 * 1024; // 128 KB of keys
// Blocks of a row that registers hold.  Against list_kernel's bins: 8 us instead of 14 for 512
// rows of up to 2048 blocks, the call 303 us instead of 386 for 384 rows of 16000 and 20.6 us
// instead of 21.3 for 8.  At 32768 (32 keys a thread, which spill) 8 rows of 16385 took 29.4 us
// instead of 20.6.
constexpr u32 kShortRow = 16384;
constexpr u32 kAbsent = 0u;           // key of a block that cannot be listed
constexpr u32 kAlways = 0xffffffffu;  // key of a block that is always listed

struct SelectArgs {
    KvView c;
    KvQuery q;
    u32 top, sink, recent;
    std::int8_t* whole;  // [seqs][heads][2 tokens][2 D]: high and low parts, down then up
    u32* keys;           // [seqs][tokens][heads][width]
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

__device__ __forceinline__ void mma16832(int (&d)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One warp per (sequence, token, head): the group's queries as whole numbers.
template <int D>
__global__ void __launch_bounds__(kQueryWarps * 32) query_kernel(const SelectArgs a)
{
    constexpr int E = D / 32;  // channels of a lane
    kv_let_next();
    const u32 heads = a.c.heads, tokens = a.q.tokens, group = a.q.group, lane = threadIdx.x & 31u;
    const u32 at = blockIdx.x * kQueryWarps + (threadIdx.x >> 5);
    if (at >= a.q.seqs * tokens * heads) return;
    const u32 h = at % heads, t = at / heads % tokens, seq = at / heads / tokens;
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
    // column 2 t: the high parts, 2 t + 1: the low ones
    std::int8_t* to = a.whole + ((static_cast<u64>(seq) * heads + h) * 2 * tokens + 2 * t) * 2 * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        to[e] = static_cast<std::int8_t>(-(-down[e] >> 7));
        to[2 * D + e] = static_cast<std::int8_t>(-(-down[e] & 127));
        to[D + e] = static_cast<std::int8_t>(up[e] >> 7);
        to[3 * D + e] = static_cast<std::int8_t>(up[e] & 127);
    }
}

// A stage of a warp's ring: the bounds of 16 blocks (a block's 64-byte pieces
// are exchanged in pairs by its number's last bit, against bank conflicts),
// their scales and whether they are there.
template <int D>
constexpr u32 kScoreStage = 16 * 2 * D + 128;
template <int D>
constexpr u32 kScoreStages = D == 256 ? 2 : 3;
template <int D>
constexpr u32 kScoreSmem = kScoreWarps * kScoreStages<D> * kScoreStage<D>;
// CTAs per SM by shared memory: about 200 KB of rings.
HD constexpr u32 score_per_sm(u32 dim) { return dim == 64 ? 3 : dim == 128 ? 2 : 1; }

template <int D>
__global__ void __launch_bounds__(kScoreWarps * 32, score_per_sm(D)) score_kernel(const SelectArgs a)
{
    constexpr u32 kChunks = D / 32;  // 64-byte pieces of a block's bounds
    constexpr u32 NS = kScoreStages<D>;
    extern __shared__ __align__(128) u8 smem[];
    __shared__ u64 line;
    kv_let_next();
    const u32 heads = a.c.heads, tokens = a.q.tokens;
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3u;
    u8* ring = smem + warp * NS * kScoreStage<D>;
    const u32 page_bytes = heads * 2 * D, page_scales = heads * 2;
    // the line of all sequences' blocks, and this CTA's share of it
    u64 all = 0;
    for (u32 s = threadIdx.x; s < a.q.seqs; s += kScoreWarps * 32) all += blocks_of_sequence(a, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (threadIdx.x == 0) line = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&line), all);
    __syncthreads();
    const u64 share = max(static_cast<u64>(kScoreShare), (line + gridDim.x - 1) / gridDim.x);
    u64 at = blockIdx.x * share;
    const u64 stop = min(at + share, line);
    u32 seq = 0, have = 0;
    u64 begin = 0;
    for (u32 base = 0; at < stop && base < a.q.seqs; base += 32) {  // the sequence that holds `at`
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
    bool queries = false;  // whether query_kernel's results may be read
    for (; at < stop; begin += have, have = ++seq < a.q.seqs ? blocks_of_sequence(a, seq) : 0) {
        const u32 first = static_cast<u32>(at - begin);
        const u32 end = static_cast<u32>(min(stop - begin, static_cast<u64>(have)));
        if (first >= end) continue;
        at = begin + end;
        const int length = kv_length(a.q.lengths, seq, a.q.width, a.c.block);
        const int* table = a.q.table + static_cast<i64>(seq) * a.q.table_stride;
        // Tasks: 16 blocks of one head, heads first, by the warps in turn.
        const u32 rows = (end - first + 15) / 16;
        const u32 skip_rows = kScoreWarps / heads, skip_heads = kScoreWarps % heads;
        auto advance = [&](u32& row, u32& h) {
            row += skip_rows;
            h += skip_heads;
            if (h >= heads) {
                h -= heads;
                ++row;
            }
        };
        auto page_of = [&](u32 row) {  // of the task's block lane % 16
            const u32 j = first + row * 16 + (lane & 15u);
            return row < rows && j < end ? kv_page(table, j, a.c.pages) : -1;
        };
        u32 issue_row = warp / heads, issue_h = warp % heads;
        int issue_page = page_of(issue_row);
        // 2 D bytes of a block: D / 8 lanes, 16 bytes each
        constexpr u32 kLanes = D / 8, kAtOnce = 32 / kLanes;
        const u32 block_at = lane / kLanes, piece = lane % kLanes;
        auto issue = [&](u32 stage) {
            const int page = issue_page;
            const u32 row = issue_row, h = issue_h;
            advance(issue_row, issue_h);
            issue_page = page_of(issue_row);
            if (row < rows) {
                u8* to = ring + stage * kScoreStage<D>;
                // a block that is not there is noted; its copy takes some page's bounds
                const u32 real = static_cast<u32>(max(page, 0));
                const u64 source = reinterpret_cast<u64>(a.c.bounds) + h * 2 * D + static_cast<u64>(real) * page_bytes;
                const u32 even = kv_shared(to) + block_at * 2 * D + ((piece >> 2) ^ (block_at & 1u)) * 64 + (piece & 3u) * 16;
#pragma unroll
                for (u32 r = 0; r < 16; r += kAtOnce) {
                    const u64 from = __shfl_sync(0xffffffffu, source, r + block_at) + piece * 16;
                    // one block at once: the pieces of odd blocks are exchanged
                    const u32 odd = kAtOnce == 1 && (r & 1u) ? 64u : 0u;
                    kv_copy16((even ^ odd) + r * 2 * D, reinterpret_cast<const void*>(from));
                }
                if (lane < 16) {
                    u32* notes = reinterpret_cast<u32*>(to + 16 * 2 * D);
                    notes[16 + lane] = page >= 0;
                    kv_copy4(notes + lane, a.c.scale + h * 2 + static_cast<u64>(real) * page_scales);
                }
            }
            kv_copy_commit();
        };
#pragma unroll
        for (u32 i = 0; i + 1 < NS; ++i) issue(i);
        if (!queries) kv_wait_before();
        queries = true;
        // Column g of a group of four tokens is the high or low part of token t0 + g / 2.  The
        // first group's stays in registers for as long as the warp's head does.
        const std::int8_t* columns = a.whole + static_cast<u64>(seq) * heads * 2 * tokens * 2 * D;
        auto column_of = [&](u32 h, u32 t0, uint4 (&y)[kChunks]) {
            const bool used = t0 + g / 2 < tokens;
            const std::int8_t* column = columns + (static_cast<u64>(h) * 2 * tokens + 2 * t0 + g) * 2 * D + c * 16;
#pragma unroll
            for (u32 k = 0; k < kChunks; ++k) {
                y[k] = make_uint4(0, 0, 0, 0);
                if (used) y[k] = *reinterpret_cast<const uint4*>(column + k * 64);
            }
        };
        uint4 y[kChunks];
        u32 y_head = heads, stage = 0;
        for (u32 row = warp / heads, h = warp % heads; row < rows; advance(row, h)) {
            kv_copy_wait<NS - 2>();
            __syncwarp();  // the stage is there, and every lane is done with the one before it
            issue(stage == 0 ? NS - 1 : stage - 1);
            const u8* tile = ring + stage * kScoreStage<D>;
            stage = stage + 1 == NS ? 0 : stage + 1;
            const u32* notes = reinterpret_cast<const u32*>(tile + 16 * 2 * D);
            const u32 j0 = first + row * 16 + g;
            const bool there0 = notes[16 + g] != 0, there1 = notes[24 + g] != 0;
            const float scale0 = __uint_as_float(notes[g]), scale1 = __uint_as_float(notes[8 + g]);
            const u8* even = tile + g * 2 * D + (g & 1u) * 64 + c * 16;  // pieces 0, 2, ..
            const u8* odd = tile + g * 2 * D + (~g & 1u) * 64 + c * 16;  // pieces 1, 3, ..
            u32* keys = a.keys + (static_cast<u64>(seq) * tokens * heads + h) * a.q.width + j0;
            for (u32 t0 = 0; t0 < tokens; t0 += 4) {
                if (t0 || y_head != h) {
                    column_of(h, t0, y);
                    y_head = tokens <= 4 ? h : heads;
                }
                int s0[4] = {0, 0, 0, 0}, s1[4] = {0, 0, 0, 0};
#pragma unroll
                for (u32 k = 0; k < kChunks; ++k) {
                    const u8* at_piece = (k & 1u ? odd : even) + (k & ~1u) * 64;
                    const uint4 x0 = *reinterpret_cast<const uint4*>(at_piece);
                    const uint4 x1 = *reinterpret_cast<const uint4*>(at_piece + 8 * 2 * D);
                    mma16832(s0, x0.x, x1.x, x0.y, x1.y, y[k].x, y[k].y);
                    mma16832(s1, x0.z, x1.z, x0.w, x1.w, y[k].z, y[k].w);
                }
                const u32 t = t0 + c;  // this lane's columns 2c and 2c + 1
                if (t < tokens) {
                    const u32 mine = blocks_of_token(length, tokens, t, a.c.block);
                    u32* to = keys + static_cast<u64>(t) * heads * a.q.width;
                    auto put = [&](u32 more, bool there, float scale, int sum) {
                        const u32 j = j0 + more;
                        u32 key = order_key(__fmul_rn(__int2float_rn(sum), scale));
                        if (j < a.sink || j + a.recent >= mine) key = kAlways;
                        if (!there || j >= mine) key = kAbsent;
                        if (j < end) to[more] = key;
                    };
                    put(0, there0, scale0, (s0[0] + s1[0]) * 128 + s0[1] + s1[1]);
                    put(8, there1, scale1, (s0[2] + s1[2]) * 128 + s0[3] + s1[3]);
                }
            }
        }
        kv_copy_wait<0>();
        __syncwarp();  // before the next sequence's copies
    }
    if (!queries) kv_wait_before();  // list_kernel waits for this kernel alone
}

// Rows of at most 32 K W blocks: a CTA of W warps per (sequence, token, head), which hold the row in
// registers, finds the key of the last block to list bit by bit; a bit costs a count and one
// barrier.
template <u32 W, int K>
__global__ void __launch_bounds__(W * 32) short_list_kernel(const SelectArgs a)
{
    __shared__ uint4 found[W];
    __shared__ u32 counts[2][W];  // of the warps, in turns
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, under = (1u << lane) - 1u;
    kv_wait_before();
    const u64 at = blockIdx.x;
    const u32 heads = a.c.heads, tokens = a.q.tokens;
    const u32 t = static_cast<u32>(at / heads % tokens), seq = static_cast<u32>(at / heads / tokens);
    const int length = kv_length(a.q.lengths, seq, a.q.width, a.c.block);
    const u32 have = blocks_of_token(length, tokens, t, a.c.block);
    // a warp's blocks: a run of whole 32s
    const u32 each = (have + W * 32 - 1) / (W * 32) * 32, from = warp * each, to = min(from + each, have);
    const u32* row = a.keys + at * a.q.width;
    u32 k[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const u32 j = from + i * 32 + lane;
        k[i] = j < to ? row[j] : kAbsent;
    }
    u32 there = 0, always = 0, least = ~0u, greatest = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        there += k[i] != kAbsent;
        always += k[i] == kAlways;
        if (k[i] != kAbsent && k[i] != kAlways) {
            least = min(least, k[i]);
            greatest = max(greatest, k[i]);
        }
    }
    there = __reduce_add_sync(0xffffffffu, there);
    always = __reduce_add_sync(0xffffffffu, always);
    least = __reduce_min_sync(0xffffffffu, least);
    greatest = __reduce_max_sync(0xffffffffu, greatest);
    if (lane == 0) found[warp] = make_uint4(there, always, least, greatest);
    __syncthreads();
    const uint4 its = lane < W ? found[lane] : make_uint4(0, 0, ~0u, 0);
    there = __reduce_add_sync(0xffffffffu, its.x);
    always = __reduce_add_sync(0xffffffffu, its.y);
    least = __reduce_min_sync(0xffffffffu, its.z);
    greatest = __reduce_max_sync(0xffffffffu, its.w);
    u32 turn = 0;
    // the sum of the counts that the first `warps` warps bring
    auto share = [&](u32 mine, u32 warps) {
        turn ^= 1u;  // the slots of the turn before may still be read
        if (lane == 0) counts[turn][warp] = mine;
        __syncthreads();
        return __reduce_add_sync(0xffffffffu, lane < warps ? counts[turn][lane] : 0);
    };
    const u32 take = min(a.top, there);
    // Listed: the keys above `limit` and the first `equals` at it.
    u32 limit = kAlways, equals = take;
    if (take == there) {
        limit = kAbsent + 1, equals = kKvAll;
    } else if (take > always) {
        auto reach = [&](u32 x) {  // keys that are x at least
            u32 n[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < K; ++i) n[i % 4] += k[i] >= x;
            return share(__reduce_add_sync(0xffffffffu, n[0] + n[1] + n[2] + n[3]), W);
        };
        const u32 differ = least ^ greatest;
        u32 bit = differ ? 0x80000000u >> __clz(static_cast<int>(differ)) : 0;
        limit = greatest & ~(bit ? 2 * bit - 1 : 0);  // the bits that all keys share
        u32 count = 0;
        for (; bit && count != take; bit >>= 1) {
            const u32 n = reach(limit | bit);
            if (n >= take) limit |= bit, count = n;
        }
        equals = count == take ? kKvAll : take - reach(limit + 1);
    }
    u32 same = 0;  // keys at the limit in front, and listed ones
    if (equals != kKvAll) {
        u32 n = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) n += k[i] == limit;
        same = share(__reduce_add_sync(0xffffffffu, n), warp);
    }
    u32 listed[K], before = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        bool chosen = k[i] >= limit;
        if (equals != kKvAll) {
            const u32 equal = __ballot_sync(0xffffffffu, k[i] == limit);
            chosen = k[i] > limit || (k[i] == limit && same + __popc(equal & under) < equals);
            same += __popc(equal);
        }
        listed[i] = __ballot_sync(0xffffffffu, chosen);
        before += __popc(listed[i]);
    }
    before = share(before, warp);
    int* list = a.blocks + at * a.top;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        if (listed[i] >> lane & 1u) list[before + __popc(listed[i] & under)] = static_cast<int>(from + i * 32 + lane);
        before += __popc(listed[i]);
    }
    for (u32 i = take + threadIdx.x; i < a.top; i += W * 32) list[i] = -1;
    if (threadIdx.x == 0) a.counts[at] = static_cast<int>(take);
}

// Any row.  `slice`: blocks of a row that one CTA of the team has.
__global__ void __launch_bounds__(1024) list_kernel(const SelectArgs a, u32 team_size, u32 slice)
{
    extern __shared__ __align__(16) u32 held[];
    __shared__ KvSelectShared sm;
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
    u32 there = 0, always = 0;  // blocks that are there, and those always listed
    u32 least = ~0u, greatest = 0;
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
    kv_gather(team, sm, least, greatest, there, always);
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
    kv_walk<false, true>(
        team, mine, equals, sm,
        [&](u32 i) -> u32 {
            const u32 k = keys[i];
            if (k == kAbsent) return 0;
            return k == kAlways || ~k < limit ? 1 : ~k == limit ? 2 : 0;
        },
        [](u32) { return 0; },
        [&](u32 i, int, bool, u32 before) {
            if (before < a.top) list[before] = static_cast<int>(first + i);
        });
    if (team.rank == 0) {
        for (u32 i = take + threadIdx.x; i < a.top; i += blockDim.x) list[i] = -1;
        if (threadIdx.x == 0) a.counts[at] = static_cast<int>(take);
    }
    kv_team_sync(team);  // nobody leaves while another may read its counts
}

u64 whole_bytes(const KvView& v, const KvQuery& q)
{
    return kv_round_up(static_cast<u64>(q.seqs) * v.heads * 2 * q.tokens * 2 * v.dim, 256);
}

u64 workspace_bytes_of(const KvView& v, const KvQuery& q)
{
    return whole_bytes(v, q) +
           kv_round_up(static_cast<u64>(q.seqs) * q.tokens * v.heads * q.width * 4, 256);
}

template <int D>
int launch(const SelectArgs& a, cudaStream_t s)
{
    static std::atomic<u64> seen{0};
    if (!kv_allow_smem(score_kernel<D>, kScoreSmem<D>, seen)) return HBFSIM_CUDA_ERROR;
    const u32 rows = a.q.seqs * a.q.tokens * a.c.heads;
    bool ok = true;
    if (a.q.width) {
        ok = kv_launch(query_kernel<D>, dim3((rows + kQueryWarps - 1) / kQueryWarps), kQueryWarps * 32, s, 0, 1, false, a);
        const u64 most = (static_cast<u64>(a.q.seqs) * a.q.width + kScoreShare - 1) / kScoreShare;
        const u32 grid = static_cast<u32>(std::min<u64>(most, static_cast<u64>(score_per_sm(D)) * kv_sm_count()));
        ok = ok && kv_launch(score_kernel<D>, dim3(grid), kScoreWarps * 32, s, kScoreSmem<D>, 1, true, a);
    }
    if (a.q.width <= kShortRow) {
        // Keys per lane against warps per barrier: 16 x 4 took 41.0 us for 512 rows of up to 2048
        // (the whole call), 8 x 8 42.2 us; 8 x 16 20.2 us for 32 rows of 4000, 16 x 8 22.1 us.
        auto* kernel = short_list_kernel<4, 4>;
        u32 warps = 4;
        if (a.q.width > 512) kernel = short_list_kernel<4, 16>;
        if (a.q.width > 2048) kernel = short_list_kernel<16, 8>, warps = 16;
        if (a.q.width > 4096) kernel = short_list_kernel<32, 8>, warps = 32;
        if (a.q.width > 8192) kernel = short_list_kernel<32, 16>, warps = 32;
        ok = ok && kv_launch(kernel, dim3(rows), warps * 32, s, 0, 1, true, a);
        return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
    }
    static std::atomic<u64> seen_list{0};
    if (!kv_allow_smem(list_kernel, kHeldKeys * 4, seen_list)) return HBFSIM_CUDA_ERROR;
    u32 team = kv_team_size(rows, a.q.width), slice = (a.q.width + team - 1) / team;
    if (slice > kHeldKeys) {  // a row that no team can hold is one CTA's
        team = 1;
        slice = a.q.width;
    }
    // many rows: small CTAs, several to an SM
    u32 threads = kv_team_threads(slice);
    if (rows > 2 * static_cast<u32>(kv_sm_count())) threads = std::min(threads, 256u);
    ok = ok && kv_launch(list_kernel, dim3(rows * team), threads, s, slice <= kHeldKeys ? slice * 4 : 0, team, true, a,
                         team, slice);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
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
    if (!blocks || !counts) return HBFSIM_INVALID_ARGUMENT;
    if (workspace_bytes < workspace_bytes_of(a.c, a.q) || (a.q.width && !workspace) ||
        !kv_aligned(workspace, 16) || !kv_aligned(blocks, 4) || !kv_aligned(counts, 4))
        return HBFSIM_INVALID_ARGUMENT;
    a.whole = static_cast<std::int8_t*>(workspace);
    a.keys = reinterpret_cast<u32*>(static_cast<u8*>(workspace) + whole_bytes(a.c, a.q));
    if (a.c.pages == 0) a.q.width = 0;  // no block is there
    a.top = top;
    a.sink = sink;
    a.recent = recent;
    a.blocks = blocks;
    a.counts = counts;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.c.dim == 64) return launch<64>(a, s);
    if (a.c.dim == 128) return launch<128>(a, s);
    return launch<256>(a, s);
}
