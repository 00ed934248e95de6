// kv_pages.cu -- who has which page of the cache (kv_v1.h): pages for new
// tokens and back, children of sequences, the pages in use moved to the front,
// and the copies that both lead to.
//
// The work is a few passes over the counts and the table, each of which needs
// all of the one before: what goes back has to be counted before free pages are
// ranked, and ranked before they are given.  The passes are device functions of
// a team of thread blocks.  A small pool is done in one launch by one of them, or for
// a resize by a cluster of up to 8 with cluster barriers between the passes; a large
// one by as many blocks as the device has SMs, a launch to a pass.  Where ranks
// count, a warp has a contiguous share, so that they are sums over the warps before
// it.
//
// Latency bounds all of it but the copies: every pass is two or three dependent reads
// and a launch or a cluster barrier of 1 to 2 us.  A resize before a decode step (64
// rows of 2,048 entries, 70,000 counts) takes 17.3 us, of a pool of 1.2 million pages
// with 510 rows of 4,096 entries 32 us for 26 MB; a compaction of such a pool 21 us
// for 31 MB (its random reads of the pages' new places are half of that), of one of
// 2,600 pages 6.6 us; a fork of 64 beams 5.3 us, of 4 documents into 256 rows of
// 16,385 entries 8.4 us for 17 MB, of 4,096 rows of 2,048 entries into as many 72 us
// for 67 MB (every old row's children are counted by going over all parents).
#include "kv.h"

namespace hbfb {
namespace {

constexpr u32 kPageThreads = 1024, kPageWarps = kPageThreads / 32;
constexpr u32 kPageTeam = 8;      // blocks of the cluster
constexpr u32 kMaxParts = 1024;   // blocks of a pass at most
constexpr u32 kDeep = 16;         // entries of a table's row that a lane has under way
// Of a resize: counts and entries that are worth a block of a cluster, and that one takes at most.  A
// cluster costs about 2 us.  Before a step of 64 rows of 2048 entries, 70,000 counts, a resize takes 17.3
// us by 8 blocks, 22.0 us by 4 and 16.9 us by a launch to a pass, which cost the host 10 us more; 200 rows
// of 190 entries (100,000 counts) 18.6 us by 8 blocks, 25.6 us by 4 and 18.9 us by a launch to a pass.
// More rows take longer by 8 blocks, a run of a row to a warp after the other: 1,024 of 128 entries 34 us
// (19 by a launch to a pass), 4,096 of 32 97 us (20), 65,536 of 2 1.3 ms (87 us); the rule does not look
// at that.
constexpr u64 kCountsEach = 16384, kEntriesEach = 16384, kCountsMost = 32768, kEntriesMost = 16384;
// Of a compaction: counts and entries that one block does alone: 4,000 of both in 8.4 us and 9.3 us by a
// launch to a pass, 8,000 in 12.8 and 10.4 us (and 5 us more of the host), 16,000 in 23.6 and 10.5 us.
constexpr u64 kCompactMost = 8192;

// The elements [from, end) of a warp.
struct Share {
    u32 from, end;
};

// The counts of a warp: a run of whole 128s (four to a lane and step).
__device__ __forceinline__ Share warp_share(u32 n, const KvTeam& team)
{
    const u32 warps = team.size * kPageWarps, warp = team.rank * kPageWarps + (threadIdx.x >> 5);
    const u64 each = (static_cast<u64>(n) + warps * 128 - 1) / (warps * 128) * 128, from = each * warp;
    return {static_cast<u32>(min(from, static_cast<u64>(n))), static_cast<u32>(min(from + each, static_cast<u64>(n)))};
}

// A lane's four counts of a step from p (a multiple of 4) on, `other` past the end.
struct Four {
    int x[4];
};
__device__ __forceinline__ Four load_four(const int* counts, u32 p, u32 end, int other)
{
    Four f;
    if (p + 4 <= end && (reinterpret_cast<std::uintptr_t>(counts) & 15) == 0) {
        const int4 y = *reinterpret_cast<const int4*>(counts + p);
        f.x[0] = y.x;
        f.x[1] = y.y;
        f.x[2] = y.z;
        f.x[3] = y.w;
    } else {
#pragma unroll
        for (u32 i = 0; i < 4; ++i) f.x[i] = p + i < end ? counts[p + i] : other;
    }
    return f;
}

__device__ __forceinline__ void store_four(int* counts, u32 p, u32 end, const Four& f)
{
    if (p + 4 <= end && (reinterpret_cast<std::uintptr_t>(counts) & 15) == 0) {
        *reinterpret_cast<int4*>(counts + p) = make_int4(f.x[0], f.x[1], f.x[2], f.x[3]);
    } else {
#pragma unroll
        for (u32 i = 0; i < 4; ++i)
            if (p + i < end) counts[p + i] = f.x[i];
    }
}

// Of four marks per lane, in order of lane and mark: how many there are before each, and in all.
struct Ranks {
    u32 before[4], all;
};
__device__ __forceinline__ Ranks rank_four(const bool (&mark)[4])
{
    const u32 lane = threadIdx.x & 31u, below = (1u << lane) - 1;
    Ranks r{{0, 0, 0, 0}, 0};
    u32 lower = 0;
#pragma unroll
    for (u32 i = 0; i < 4; ++i) {
        const u32 who = __ballot_sync(0xffffffffu, mark[i]);
        lower += __popc(who & below);
        r.all += __popc(who);
    }
#pragma unroll
    for (u32 i = 0; i < 4; ++i) {
        r.before[i] = lower;
        lower += mark[i];
    }
    return r;
}

// How many of a warp's counts are marked.
template <typename Mark>
__device__ __forceinline__ u32 count_marked(const int* counts, u32 n, const KvTeam& team, int other, const Mark& mark)
{
    const Share own = warp_share(n, team);
    u32 sum = 0;
#pragma unroll 4
    for (u32 p = own.from + (threadIdx.x & 31u) * 4; p < own.end; p += 128) {
        const Four f = load_four(counts, p, own.end, other);
#pragma unroll
        for (u32 i = 0; i < 4; ++i) sum += mark(f.x[i]);
    }
    return __reduce_add_sync(0xffffffffu, sum);
}

// Sums over the block, by every thread.
template <u32 N>
__device__ __forceinline__ void block_sums(u32 (&x)[N], u32 (*warp_sums)[kPageWarps])
{
    const u32 lane = threadIdx.x & 31u;
#pragma unroll
    for (u32 k = 0; k < N; ++k) x[k] = __reduce_add_sync(0xffffffffu, x[k]);
    __syncthreads();  // earlier readers of warp_sums are done
    if (lane == 0) {
#pragma unroll
        for (u32 k = 0; k < N; ++k) warp_sums[k][threadIdx.x >> 5] = x[k];
    }
    __syncthreads();
#pragma unroll
    for (u32 k = 0; k < N; ++k) x[k] = __reduce_add_sync(0xffffffffu, warp_sums[k][lane]);
}

// Sums of the parts of earlier warps (of every block) and of all; of other parts, if given, of all.
// begin() asks for them, end() adds them up.
struct Before {
    u32 mine, all, others;
    u32 inside, x[3];

    __device__ __forceinline__ void begin(const u32* parts, const KvTeam& team, const u32* more = nullptr)
    {
        const u32 lane = threadIdx.x & 31u, own = team.rank * kPageWarps, n = team.size * kPageWarps;
        inside = lane < threadIdx.x >> 5 ? parts[own + lane] : 0;
        x[0] = x[1] = x[2] = 0;
        for (u32 i = threadIdx.x; i < n; i += kPageThreads) {
            const u32 part = parts[i];
            x[1] += part;
            if (i < own) x[0] += part;
            if (more) x[2] += more[i];
        }
    }
    __device__ __forceinline__ void end(u32 (*warp_sums)[kPageWarps])
    {
        block_sums(x, warp_sums);
        mine = x[0] + __reduce_add_sync(0xffffffffu, inside);
        all = x[1];
        others = x[2];
    }
};

// Calls run(row, from, end) for runs of a table's rows, up to 32 * Deep entries to a warp; the
// blocks of a team take them in turn, so that few runs are spread over all of them.
template <u32 Deep, typename Run>
__device__ __forceinline__ void for_runs(u32 rows, u32 width, const KvTeam& team, const Run& run)
{
    const u32 per_row = (width + 32 * Deep - 1) / (32 * Deep);
    const u64 units = static_cast<u64>(rows) * per_row;
    for (u64 u = (threadIdx.x >> 5) * team.size + team.rank; u < units; u += team.size * kPageWarps) {
        const u32 row = static_cast<u32>(u / per_row);
        const u32 from = static_cast<u32>(u - static_cast<u64>(row) * per_row) * 32 * Deep;
        run(row, from, min(from + 32 * Deep, width));
    }
}

// A lane's entries of a run, all under way at once: from[first + lane + 32 i], -1 past the end.
template <u32 Deep>
__device__ __forceinline__ void load_run(const int* from, u32 first, u32 end, int (&e)[Deep])
{
    const u32 lane = threadIdx.x & 31u;
#pragma unroll
    for (u32 i = 0; i < Deep; ++i) e[i] = first + lane + 32 * i < end ? from[first + lane + 32 * i] : -1;
}

// The counts of a pool into their new place.
__device__ __forceinline__ void copy_counts(const int* from, int* to, u32 n, const KvTeam& team)
{
    if (from == to) return;
    const Share own = warp_share(n, team);
#pragma unroll 1
    for (u32 p = own.from + (threadIdx.x & 31u) * 4; p < own.end; p += 512) {
        Four f[4];
#pragma unroll
        for (u32 i = 0; i < 4; ++i) f[i] = load_four(from, p + 128 * i, own.end, 0);
#pragma unroll
        for (u32 i = 0; i < 4; ++i) store_four(to, p + 128 * i, own.end, f[i]);
    }
}

// ---------------------------------------------------------------------------
// Pages for new tokens and back

struct ResizeArgs {
    const int* refs;
    const int* table;
    i64 table_stride;
    const int* lengths;
    const int* want;
    const int* freed;
    const int* freed_counts;
    int* refs_out;
    int* table_out;
    i64 table_out_stride;
    int* limits;
    int* src;
    int* dst;
    u32 seqs, width, block, freed_rows, freed_width, pages;
    // workspace
    u32* free_part;   // [blocks][kPageWarps] free pages of a warp's share
    u32* asked_part;  // [blocks][kPageWarps] asked blocks of a warp's runs
    u32* claim_part;  // [blocks][kPageWarps] claims of a warp's runs
    u32* free_all;    // free pages
    int* claims;      // [pages] of a shared page: how often it is asked for
    int* last;        // [pages] and by which sequence last
    int* pool;        // the first free pages in ascending order
    u8* state;        // [seqs][width] what becomes of an asked block
};
enum State : u32 { kKeep = 0, kNew = 1, kPart = 2, kStays = 3 };

struct Row {
    u32 held, goal, first, need;  // tokens; asked blocks [first, need) if goal > held
};
__device__ __forceinline__ Row row_of(const ResizeArgs& a, u32 s)
{
    Row r;
    r.held = static_cast<u32>(kv_length(a.lengths, s, a.width, a.block));
    r.goal = static_cast<u32>(kv_length(a.want, s, a.width, a.block));
    r.first = r.held / a.block;
    r.need = (r.goal + a.block - 1) / a.block;
    return r;
}

// Runs of the table's rows that are a warp's, in order: [from, end).
struct Runs {
    u64 from, end;
    u32 per_row;
};
__device__ __forceinline__ Runs runs_of(const ResizeArgs& a, const KvTeam& team)
{
    const u32 per_row = (a.width + 32 * kDeep - 1) / (32 * kDeep);
    const u64 units = static_cast<u64>(a.seqs) * per_row, warps = team.size * kPageWarps;
    const u64 warp = team.rank * kPageWarps + (threadIdx.x >> 5);
    const u64 each = (units + warps - 1) / warps;
    return {min(each * warp, units), min(each * (warp + 1), units), per_row};
}

// A run: entries [first, end) of a row, of which blocks [from, to) are asked for.
struct Run {
    u32 seq, first, end, from, to;
    Row row;
    const int* in;
    int* out;
    u8* state;

    __device__ __forceinline__ Run(const ResizeArgs& a, const Runs& runs, u64 u)
    {
        seq = static_cast<u32>(u / runs.per_row);
        first = static_cast<u32>(u - static_cast<u64>(seq) * runs.per_row) * 32 * kDeep;
        end = min(first + 32 * kDeep, a.width);
        row = row_of(a, seq);
        from = max(first, row.first);
        to = row.goal > row.held ? min(row.need, end) : 0;
        in = a.table + static_cast<i64>(seq) * a.table_stride;
        out = a.table_out + static_cast<i64>(seq) * a.table_out_stride;
        state = a.state + static_cast<u64>(seq) * a.width;
    }
};
// The asked blocks of a warp's runs, in order, 128 at a time: asked(run, j), where the lane's blocks
// are j + 32 i, i < kStep, as far as they lie before run.to.  Most runs of a decode step ask for none,
// those of a prompt for all: loops of a few loads each keep the instructions few, which bound a
// cluster's 8 SMs.
constexpr u32 kStep = 4;
template <typename Asked>
__device__ __forceinline__ void for_asked(const ResizeArgs& a, const KvTeam& team, const Asked& asked)
{
    const Runs runs = runs_of(a, team);
#pragma unroll 1
    for (u64 u = runs.from; u < runs.end; ++u) {
        const Run run(a, runs, u);
#pragma unroll 1
        for (u32 j = run.from; j < run.to; j += 32 * kStep) asked(run, j + (threadIdx.x & 31u));
    }
}

// Counts into their new place.
__device__ void resize_begin(const ResizeArgs& a, const KvTeam& team)
{
    copy_counts(a.refs, a.refs_out, a.pages, team);
    const u32 threads = team.size * blockDim.x;
    for (u32 s = team.rank * blockDim.x + threadIdx.x; s < a.seqs; s += threads) {
        a.limits[s] = static_cast<int>(row_of(a, s).goal);
        a.src[s] = a.dst[s] = -1;
    }
}

// What lies behind the rows' new ends goes back.
__device__ __forceinline__ void resize_rows(const ResizeArgs& a, const KvTeam& team)
{
    const u32 lane = threadIdx.x & 31u;
    const bool apart = a.table_out != a.table;
    const Runs runs = runs_of(a, team);
    for (u64 u = runs.from; u < runs.end; ++u) {
        const Run run(a, runs, u);
        const bool still = run.end <= run.row.need && run.from >= run.to;  // nothing happens to these
        if (still && !apart) continue;
        int e[kDeep];
        load_run(run.in, run.first, run.end, e);
        if (still) {
#pragma unroll
            for (u32 i = 0; i < kDeep; ++i)
                if (run.first + lane + 32 * i < run.end) run.out[run.first + lane + 32 * i] = e[i];
            continue;
        }
#pragma unroll
        for (u32 i = 0; i < kDeep; ++i) {
            const u32 j = run.first + lane + 32 * i;
            const bool there = static_cast<u32>(e[i]) < a.pages, behind = j >= run.row.need;
            if (there && behind) atomicSub(a.refs_out + e[i], 1);
            if (there && j >= run.from && j < run.to) {  // asked for: counted in the next pass
                a.claims[e[i]] = 0;
                a.last[e[i]] = -1;
            }
            if (j < run.end && (apart || (behind && e[i] != -1))) run.out[j] = behind ? -1 : e[i];
        }
    }
}

// And what an eviction freed.
__device__ void give_back_listed(const ResizeArgs& a, const KvTeam& team)
{
    for (u32 r = (threadIdx.x >> 5) * team.size + team.rank; r < a.freed_rows; r += team.size * kPageWarps) {
        const int* list = a.freed + static_cast<u64>(r) * a.freed_width;
        const u32 end = min(static_cast<u32>(max(a.freed_counts[r], 0)), a.freed_width);
#pragma unroll 1
        for (u32 j = 0; j < end; j += 128) {
            int e[4];
            load_run(list, j, end, e);
#pragma unroll
            for (u32 i = 0; i < 4; ++i)
                if (static_cast<u32>(e[i]) < a.pages) atomicSub(a.refs_out + e[i], 1);
        }
    }
}

__device__ void resize_back(const ResizeArgs& a, const KvTeam& team)
{
    resize_rows(a, team);
    give_back_listed(a, team);
}

// How often shared pages are asked for, and how many are free.
__device__ void resize_count(const ResizeArgs& a, const KvTeam& team)
{
    u32 asked = 0;
    for_asked(a, team, [&](const Run& run, u32 j) {
        int e[kStep], count[kStep];
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) {
            asked += j + 32 * i < run.to;
            e[i] = j + 32 * i < run.to ? run.out[j + 32 * i] : -1;
        }
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) count[i] = static_cast<u32>(e[i]) < a.pages ? a.refs_out[e[i]] : 0;
#pragma unroll
        for (u32 i = 0; i < kStep; ++i)
            if (count[i] > 1) {
                atomicAdd(a.claims + e[i], 1);
                atomicMax(a.last + e[i], static_cast<int>(run.seq));
            }
    });
    const u32 free = count_marked(a.refs_out, a.pages, team, 1, [](int x) { return x < 1; });
    asked = __reduce_add_sync(0xffffffffu, asked);
    if ((threadIdx.x & 31u) == 0) {
        a.free_part[team.rank * kPageWarps + (threadIdx.x >> 5)] = free;
        a.asked_part[team.rank * kPageWarps + (threadIdx.x >> 5)] = asked;
    }
}

// What becomes of the asked blocks; the free pages in ascending order, as many as may be asked for.
__device__ void resize_rank(const ResizeArgs& a, const KvTeam& team, u32 (*warp_sums)[kPageWarps])
{
    u32 claims = 0;
    Before before;
    before.begin(a.free_part, team, a.asked_part);
    // the first of the warp's counts, on their way while the asked blocks are looked at
    const Share own = warp_share(a.pages, team);
    Four f[4];
    auto load_counts = [&](u32 p0) {
#pragma unroll
        for (u32 k = 0; k < 4; ++k) f[k] = load_four(a.refs_out, p0 + 128 * k + (threadIdx.x & 31u) * 4, own.end, 1);
    };
    load_counts(own.from);
    for_asked(a, team, [&](const Run& run, u32 j) {
        int e[kStep], count[kStep];
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) e[i] = j + 32 * i < run.to ? run.out[j + 32 * i] : -1;
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) count[i] = static_cast<u32>(e[i]) < a.pages ? a.refs_out[e[i]] : 0;
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) {
            if (j + 32 * i >= run.to) break;
            State state = static_cast<u32>(e[i]) < a.pages ? kKeep : kNew;
            if (count[i] > 1)
                state = a.claims[e[i]] >= count[i] && a.last[e[i]] == static_cast<int>(run.seq) ? kStays : kPart;
            run.state[j + 32 * i] = static_cast<u8>(state);
            claims += state == kNew || state == kPart;
        }
    });
    claims = __reduce_add_sync(0xffffffffu, claims);
    if ((threadIdx.x & 31u) == 0) a.claim_part[team.rank * kPageWarps + (threadIdx.x >> 5)] = claims;
    before.end(warp_sums);
    if (team.rank == 0 && threadIdx.x == 0) *a.free_all = before.all;
    u32 rank = before.mine;
#pragma unroll 1
    for (u32 p0 = own.from; p0 < own.end && rank < before.others; p0 += 512) {
        const u32 p = p0 + (threadIdx.x & 31u) * 4;
        if (p0 != own.from) load_counts(p0);
#pragma unroll
        for (u32 k = 0; k < 4; ++k) {
            const bool free[4] = {f[k].x[0] < 1, f[k].x[1] < 1, f[k].x[2] < 1, f[k].x[3] < 1};
            const Ranks r = rank_four(free);
#pragma unroll
            for (u32 i = 0; i < 4; ++i)
                if (free[i] && rank + r.before[i] < before.others)
                    a.pool[rank + r.before[i]] = static_cast<int>(p + 128 * k + i);
            rank += r.all;
        }
    }
}

// Claims get their pages.
__device__ void resize_give(const ResizeArgs& a, const KvTeam& team, u32 (*warp_sums)[kPageWarps])
{
    const u32 lane = threadIdx.x & 31u, free = *a.free_all;
    Before claims_before;
    claims_before.begin(a.claim_part, team);
    claims_before.end(warp_sums);
    u32 rank = claims_before.mine;
    for_asked(a, team, [&](const Run& run, u32 j) {
        u32 state[kStep], before[kStep];
        int page[kStep];
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) state[i] = j + 32 * i < run.to ? run.state[j + 32 * i] : kKeep;
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) {
            const bool claim = state[i] == kNew || state[i] == kPart;
            const u32 who = __ballot_sync(0xffffffffu, claim);
            before[i] = rank + __popc(who & ((1u << lane) - 1));
            rank += __popc(who);
            page[i] = claim && before[i] < free ? a.pool[before[i]] : -1;
        }
#pragma unroll
        for (u32 i = 0; i < kStep; ++i) {
            if (state[i] == kKeep) continue;
            const u32 block = j + 32 * i;
            if (state[i] == kStays ? before[i] > free : page[i] < 0) {  // not served
                atomicMin(a.limits + run.seq, static_cast<int>(max(run.row.held, block * a.block)));
            } else if (state[i] != kStays) {
                if (state[i] == kPart) {
                    const int old = run.out[block];
                    atomicSub(a.refs_out + old, 1);
                    if (block == run.row.first && run.row.held % a.block) {
                        a.src[run.seq] = old;
                        a.dst[run.seq] = page[i];
                    }
                }
                a.refs_out[page[i]] = 1;
                run.out[block] = page[i];
            }
        }
    });
}

__global__ void __launch_bounds__(kPageThreads) resize_cluster_kernel(const ResizeArgs a)
{
    __shared__ u32 warp_sums[3][kPageWarps];
    const KvTeam team{blockIdx.x, gridDim.x};
    resize_begin(a, team);
    if (a.refs_out != a.refs) kv_team_sync(team);
    resize_back(a, team);
    kv_team_sync(team);
    resize_count(a, team);
    kv_team_sync(team);
    resize_rank(a, team, warp_sums);
    kv_team_sync(team);
    resize_give(a, team, warp_sums);
}

template <int kPass>
__global__ void __launch_bounds__(kPageThreads) resize_pass_kernel(const ResizeArgs a)
{
    __shared__ u32 warp_sums[3][kPageWarps];
    kv_let_next();
    kv_wait_before();
    const KvTeam team{blockIdx.x, gridDim.x};
    if constexpr (kPass == 0 || kPass == 5) resize_begin(a, team);
    if constexpr (kPass == 1 || kPass == 5) resize_back(a, team);
    if constexpr (kPass == 2) resize_count(a, team);
    if constexpr (kPass == 3) resize_rank(a, team, warp_sums);
    if constexpr (kPass == 4) resize_give(a, team, warp_sums);
}

// ---------------------------------------------------------------------------
// Children

struct ForkArgs {
    const int* refs;
    const int* table;
    i64 table_stride;
    const int* lengths;
    const int* parents;
    int* refs_out;
    int* table_out;
    int* lengths_out;
    u32 seqs, rows, width, block, pages;
};

__device__ __forceinline__ u32 blocks_held(const ForkArgs& a, u32 s)
{
    return (static_cast<u32>(kv_length(a.lengths, s, a.width, a.block)) + a.block - 1) / a.block;
}

// The new rows.
__device__ void fork_rows(const ForkArgs& a, const KvTeam& team)
{
    const u32 lane = threadIdx.x & 31u, threads = team.size * blockDim.x;
    copy_counts(a.refs, a.refs_out, a.pages, team);
    for (u32 r = team.rank * blockDim.x + threadIdx.x; r < a.rows; r += threads) {
        const u32 parent = static_cast<u32>(a.parents[r]);
        a.lengths_out[r] = parent < a.seqs ? kv_length(a.lengths, parent, a.width, a.block) : 0;
    }
    for_runs<8>(a.rows, a.width, team, [&](u32 r, u32 first, u32 end) {
        const u32 parent = static_cast<u32>(a.parents[r]);
        const u32 blocks = parent < a.seqs ? blocks_held(a, parent) : 0;
        const int* from = a.table + static_cast<i64>(parent < a.seqs ? parent : 0) * a.table_stride;
        int* to = a.table_out + static_cast<u64>(r) * a.width;
        int e[8];
        load_run(from, first, min(end, blocks), e);
#pragma unroll
        for (u32 i = 0; i < 8; ++i)
            if (first + lane + 32 * i < end) to[first + lane + 32 * i] = e[i];
    });
}

// Pages are counted for every child that goes on from an old row, less the row itself.
__device__ void fork_count(const ForkArgs& a, const KvTeam& team)
{
    const u32 lane = threadIdx.x & 31u;
    for_runs<4>(a.seqs, a.width, team, [&](u32 s, u32 first, u32 end) {
        int e[4];
        load_run(a.table + static_cast<i64>(s) * a.table_stride, first, end, e);
        const u32 blocks = blocks_held(a, s);
        u32 children = 0;
#pragma unroll 8
        for (u32 r = lane; r < a.rows; r += 32) children += a.parents[r] == static_cast<int>(s);
        children = __reduce_add_sync(0xffffffffu, children);
#pragma unroll
        for (u32 i = 0; i < 4; ++i) {
            const int by = first + lane + 32 * i < blocks ? static_cast<int>(children) - 1 : -1;
            if (by != 0 && static_cast<u32>(e[i]) < a.pages) atomicAdd(a.refs_out + e[i], by);
        }
    });
}

template <int kPass>
__global__ void __launch_bounds__(kPageThreads, 2) fork_pass_kernel(const ForkArgs a)
{
    kv_let_next();
    kv_wait_before();
    const KvTeam team{blockIdx.x, gridDim.x};
    if constexpr (kPass != 1) fork_rows(a, team);
    if constexpr (kPass != 0) fork_count(a, team);
}

// ---------------------------------------------------------------------------
// Pages in use to the front

struct CompactArgs {
    const int* refs;
    const int* table;
    i64 table_stride;
    int* refs_out;
    int* table_out;
    i64 table_out_stride;
    int* src;
    int* dst;
    int* live;
    int* where;
    u32 seqs, width, pages;
    u32* live_part;  // workspace: [blocks][kPageWarps] pages in use of a warp's share
};

__device__ void compact_count(const CompactArgs& a, const KvTeam& team)
{
    const u32 live = count_marked(a.refs, a.pages, team, 0, [](int x) { return x > 0; });
    if ((threadIdx.x & 31u) == 0) a.live_part[team.rank * kPageWarps + (threadIdx.x >> 5)] = live;
    const u32 threads = team.size * blockDim.x, room = a.pages / 2;
    for (u32 i = team.rank * blockDim.x + threadIdx.x; i < room; i += threads) a.src[i] = a.dst[i] = -1;
}

// The moves: page p in use past the n that are has n - (pages in use up to p) such pages above it,
// free page p below has p - (pages in use before p) free ones below it.  Until the next pass, `where`
// holds -2 - move of a page that moves.
__device__ void compact_rank(const CompactArgs& a, const KvTeam& team, u32 (*warp_sums)[kPageWarps])
{
    Before before;
    before.begin(a.live_part, team);
    before.end(warp_sums);
    const u32 n = before.all;
    if (team.rank == 0 && threadIdx.x == 0) *a.live = static_cast<int>(n);
    const Share own = warp_share(a.pages, team);
    u32 rank = before.mine;
#pragma unroll 1
    for (u32 p0 = own.from; p0 < own.end; p0 += 256) {
        Four f[2];
#pragma unroll
        for (u32 k = 0; k < 2; ++k) f[k] = load_four(a.refs, p0 + 128 * k + (threadIdx.x & 31u) * 4, own.end, 0);
#pragma unroll
        for (u32 k = 0; k < 2; ++k) {
            const u32 first = p0 + 128 * k + (threadIdx.x & 31u) * 4;
            const bool live[4] = {f[k].x[0] > 0, f[k].x[1] > 0, f[k].x[2] > 0, f[k].x[3] > 0};
            const Ranks r = rank_four(live);
            Four place;
#pragma unroll
            for (u32 i = 0; i < 4; ++i) {
                const u32 p = first + i, earlier = rank + r.before[i];  // pages in use before p
                place.x[i] = -1;
                if (p >= own.end) continue;
                if (p < n) {
                    if (live[i]) {
                        place.x[i] = static_cast<int>(p);
                        if (a.refs_out != a.refs) a.refs_out[p] = f[k].x[i];
                    } else {
                        a.dst[p - earlier] = static_cast<int>(p);  // its count comes with the page
                    }
                } else if (live[i]) {
                    const u32 move = n - 1 - earlier;
                    a.src[move] = static_cast<int>(p);
                    place.x[i] = -2 - static_cast<int>(move);  // its count leaves with the page
                } else {
                    a.refs_out[p] = 0;
                }
            }
            if (first < own.end) store_four(a.where, first, own.end, place);
            rank += r.all;
        }
    }
}

__device__ void compact_move(const CompactArgs& a, const KvTeam& team)
{
    const u32 lane = threadIdx.x & 31u, threads = team.size * blockDim.x, room = a.pages / 2;
    // entries: a page that moves is found by its number or, if the loop below was faster, by its place
    for_runs<8>(a.seqs, a.width, team, [&](u32 s, u32 first, u32 end) {
        int* to = a.table_out + static_cast<i64>(s) * a.table_out_stride;
        int e[8];
        bool there[8];
        load_run(a.table + static_cast<i64>(s) * a.table_stride, first, end, e);
#pragma unroll
        for (u32 i = 0; i < 8; ++i) {
            there[i] = static_cast<u32>(e[i]) < a.pages;
            if (there[i]) e[i] = *static_cast<volatile int*>(a.where + e[i]);
        }
#pragma unroll
        for (u32 i = 0; i < 8; ++i) {
            if (there[i] && e[i] < -1) e[i] = a.dst[-2 - e[i]];
            if (first + lane + 32 * i < end) to[first + lane + 32 * i] = e[i];
        }
    });
    for (u32 i = team.rank * blockDim.x + threadIdx.x; i < room; i += threads) {
        const int from = a.src[i];
        if (from < 0) break;  // moves are listed without gaps
        const int to = a.dst[i], count = a.refs[from];
        a.refs_out[to] = count;
        a.refs_out[from] = 0;
        *static_cast<volatile int*>(a.where + from) = to;
    }
}

__global__ void __launch_bounds__(kPageThreads) compact_small_kernel(const CompactArgs a)
{
    __shared__ u32 sm[3][kPageWarps];
    const KvTeam team{blockIdx.x, gridDim.x};
    compact_count(a, team);
    kv_team_sync(team);
    compact_rank(a, team, sm);
    kv_team_sync(team);
    compact_move(a, team);
}

template <int kPass>
__global__ void __launch_bounds__(kPageThreads, 2) compact_pass_kernel(const CompactArgs a)
{
    __shared__ u32 sm[3][kPageWarps];
    kv_let_next();
    kv_wait_before();
    const KvTeam team{blockIdx.x, gridDim.x};
    if constexpr (kPass == 0) compact_count(a, team);
    else if constexpr (kPass == 1) compact_rank(a, team, sm);
    else compact_move(a, team);
}

// ---------------------------------------------------------------------------
// Copies

// A page's data in pieces of 16 KB, eight loads of a thread under way, and no more thread blocks than
// there are pieces: the hardware hands them out (a gigabyte of 32 KB pages takes 307 us, 97 % of a copy's
// rate; a grid that stays and strides over the pieces took 330 to 360 us, pieces of 32 KB by 512 threads
// 351 us).  Lists kept at capacity are mostly empty: long ones go by up to 32 moves to a thread block, which
// costs a few per cent where they are full (groups of 6: 319 us).  600,000 entries of such pages take 40
// us with no move among them, 63 us with 1,000 (floor 11), 152 us with 9,000 (floor 96); 10,000 entries
// with none 12 us.
constexpr u32 kCopyThreads = 128, kCopyDeep = 8, kCopyGroup = 32;
constexpr u32 kCopyPiece = kCopyThreads * kCopyDeep * 16;  // bytes of a thread block at a time

struct CopyArgs {
    KvView from, to;
    const int* src;
    const int* dst;
    u64 count, groups;
    u32 group;     // moves of a thread block
    u32 per_page;  // pieces of a page's data; its scales and bounds go with the first
    u64 page_bytes;
};

__device__ __forceinline__ uint4 load_once(const uint4* from)
{
    uint4 x;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "l"(from)
                 : "memory");
    return x;
}

// A piece of page `src` to page `dst`.
__device__ __forceinline__ void copy_piece(const CopyArgs& a, u32 src, u32 dst, u32 part)
{
    const u64 first = static_cast<u64>(part) * kCopyPiece;
    const uint4* from = reinterpret_cast<const uint4*>(a.from.data + src * a.page_bytes + first) + threadIdx.x;
    uint4* to = reinterpret_cast<uint4*>(a.to.data + dst * a.page_bytes + first) + threadIdx.x;
    const u32 left = static_cast<u32>(min(a.page_bytes - first, static_cast<u64>(kCopyPiece))) / 16;
    uint4 x[kCopyDeep];
#pragma unroll
    for (u32 i = 0; i < kCopyDeep; ++i)
        if (threadIdx.x + i * kCopyThreads < left) x[i] = load_once(from + i * kCopyThreads);
    if (part == 0) {
        const u32 bounds = a.from.heads * 2 * a.from.dim / 16, scales = a.from.heads;  // of 16 and of 8 bytes
        const uint4* b = reinterpret_cast<const uint4*>(a.from.bounds) + static_cast<u64>(src) * bounds;
        uint4* b_to = reinterpret_cast<uint4*>(a.to.bounds) + static_cast<u64>(dst) * bounds;
        for (u32 i = threadIdx.x; i < bounds; i += kCopyThreads) b_to[i] = b[i];
        const float2* s = reinterpret_cast<const float2*>(a.from.scale) + static_cast<u64>(src) * scales;
        float2* s_to = reinterpret_cast<float2*>(a.to.scale) + static_cast<u64>(dst) * scales;
        for (u32 i = threadIdx.x; i < scales; i += kCopyThreads) s_to[i] = s[i];
    }
#pragma unroll
    for (u32 i = 0; i < kCopyDeep; ++i)
        if (threadIdx.x + i * kCopyThreads < left) to[i * kCopyThreads] = x[i];
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const CopyArgs a)
{
    const u32 lane = threadIdx.x & 31u;
    for (u64 unit = blockIdx.x; unit < a.groups * a.per_page; unit += gridDim.x) {
        const u64 group = unit / a.per_page, move = group * a.group + lane;
        const u32 part = static_cast<u32>(unit - group * a.per_page);
        const bool listed = lane < a.group && move < a.count;
        const u32 page = listed ? static_cast<u32>(a.src[move]) : ~0u;
        const u32 page_to = listed ? static_cast<u32>(a.dst[move]) : ~0u;
        u32 left_moves = __ballot_sync(0xffffffffu, page < a.from.pages && page_to < a.to.pages);
        for (; left_moves; left_moves &= left_moves - 1) {
            const int which = __ffs(left_moves) - 1;
            copy_piece(a, __shfl_sync(0xffffffffu, page, which), __shfl_sync(0xffffffffu, page_to, which), part);
        }
    }
}

// ---------------------------------------------------------------------------

bool table_fits(u64 rows, u64 width) { return rows * width <= 0x7fffffffull; }

// Takes parts of a workspace one after the other, 256 bytes aligned.
struct Room {
    u64 at = 0;
    u64 take(u64 bytes)
    {
        const u64 here = at;
        at += kv_round_up(bytes, 256);
        return here;
    }
};

// Thread blocks of a pass.
u32 pass_blocks()
{
    return std::min<u32>(kMaxParts, static_cast<u32>(kv_sm_count()));
}

// A count for every warp of a pass or a cluster.
u64 part_bytes() { return kv_round_up(u64{std::max(pass_blocks(), kPageTeam)} * kPageWarps * 4, 256); }

struct ResizeRoom {
    u64 free_part, asked_part, claim_part, free_all, claims, last, pool, state, bytes;
};
ResizeRoom resize_room(const hbfsim_kv_resize_batch_v1& b)
{
    Room room;
    ResizeRoom r{};
    r.free_part = room.take(part_bytes());
    r.asked_part = room.take(part_bytes());
    r.claim_part = room.take(part_bytes());
    r.free_all = room.take(4);
    r.claims = room.take(b.pages * 4);
    r.last = room.take(b.pages * 4);
    r.pool = room.take(std::min(b.pages, u64{b.seqs} * b.width) * 4);
    r.state = room.take(u64{b.seqs} * b.width);
    r.bytes = room.at;
    return r;
}

int resize_check(const hbfsim_kv_resize_batch_v1* b)
{
    if (!b || b->struct_size != sizeof(*b) || b->version != HBFSIM_KV_V1_VERSION || b->reserved)
        return HBFSIM_INVALID_ARGUMENT;
    if (b->block_tokens != 16 && b->block_tokens != 32 && b->block_tokens != 64) return HBFSIM_UNSUPPORTED;
    if (b->seqs > kKvMaxSeqs || b->width > kKvMaxWidth || b->pages > 0x7fffffffull ||
        u64{b->width} * b->block_tokens > 0x7fffffffull || !table_fits(b->seqs, b->width) ||
        !table_fits(b->freed_rows, b->freed_width))
        return HBFSIM_INVALID_ARGUMENT;
    return HBFSIM_OK;
}

// Launches a pass over so many blocks, set up behind the one before.
template <typename Args>
bool pass(void (*kernel)(Args), u32 blocks, bool behind, const Args& a, cudaStream_t s)
{
    return kv_launch(kernel, dim3(blocks), kPageThreads, s, 0, 1, behind, a);
}

template <typename Args>
bool cluster(void (*kernel)(Args), u32 team, const Args& a, cudaStream_t s)
{
    return kv_launch(kernel, dim3(team), kPageThreads, s, 0, team, false, a);
}

// Blocks of a cluster that does `counts` counts and `entries` entries in one launch; 0: too much for
// it.  The entries of an eviction's lists are not counted: few of their places are taken.
// `runs`: of rows, a warp each.
u32 cluster_size(u64 counts, u64 entries, u64 runs)
{
    u32 team = 1;
    while (team < kPageTeam &&
           (counts > team * kCountsEach || entries > team * kEntriesEach || runs > team * kPageWarps))
        team *= 2;
    return counts > kPageTeam * kCountsMost || entries > team * kEntriesMost ? 0 : team;
}


}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" uint64_t hbfsim_kv_resize_workspace_v1(const hbfsim_kv_resize_batch_v1* b)
{
    return resize_check(b) == HBFSIM_OK ? resize_room(*b).bytes : 0;
}

extern "C" int hbfsim_kv_resize_v1(const hbfsim_kv_resize_batch_v1* b, void* stream)
{
    if (const int rc = resize_check(b)) return rc;
    if (b->seqs == 0 && b->freed_rows == 0 && b->refs_out == b->refs) return HBFSIM_OK;
    const u64 entries = u64{b->seqs} * b->width, listed = u64{b->freed_rows} * b->freed_width;
    if ((b->pages && (!b->refs || !b->refs_out)) || (entries && (!b->table || !b->table_out)) ||
        (b->seqs && (!b->lengths || !b->want || !b->limits || !b->src || !b->dst)) ||
        (listed && (!b->freed || !b->freed_counts)) || !b->workspace)
        return HBFSIM_INVALID_ARGUMENT;
    for (const void* p : {static_cast<const void*>(b->refs), static_cast<const void*>(b->table),
                          static_cast<const void*>(b->lengths), static_cast<const void*>(b->want),
                          static_cast<const void*>(b->freed), static_cast<const void*>(b->freed_counts),
                          static_cast<const void*>(b->refs_out), static_cast<const void*>(b->table_out),
                          static_cast<const void*>(b->limits), static_cast<const void*>(b->src),
                          static_cast<const void*>(b->dst)})
        if (!kv_aligned(p, 4)) return HBFSIM_INVALID_ARGUMENT;
    const ResizeRoom room = resize_room(*b);
    if (!kv_aligned(b->workspace, 16) || b->workspace_bytes < room.bytes) return HBFSIM_INVALID_ARGUMENT;
    if (entries && b->table_out == b->table && b->table_out_stride != b->table_stride) return HBFSIM_INVALID_ARGUMENT;
    // rows of an output may not lie in one another
    if (b->seqs > 1 && std::abs(b->table_out_stride) < static_cast<i64>(b->width)) return HBFSIM_INVALID_ARGUMENT;
    const KvExtent out[] = {{b->refs_out, b->pages * 4},
                          {b->table_out, b->seqs, b->width, b->table_out_stride},
                          {b->limits, u64{b->seqs} * 4},
                          {b->src, u64{b->seqs} * 4},
                          {b->dst, u64{b->seqs} * 4},
                          {b->workspace, room.bytes}};
    const KvExtent in[] = {{b->refs, b->pages * 4},          {b->table, b->seqs, b->width, b->table_stride},
                         {b->lengths, u64{b->seqs} * 4},   {b->want, u64{b->seqs} * 4},
                         {b->freed, listed * 4},           {b->freed_counts, u64{b->freed_rows} * 4}};
    if (kv_would_race(out, in, {0, 1, -1, -1, -1, -1})) return HBFSIM_INVALID_ARGUMENT;
    u8* w = static_cast<u8*>(b->workspace);
    const ResizeArgs a{b->refs, b->table, b->table_stride, b->lengths, b->want, b->freed, b->freed_counts,
                       b->refs_out, b->table_out, b->table_out_stride, b->limits, b->src, b->dst, b->seqs, b->width,
                       b->block_tokens, listed ? b->freed_rows : 0, b->freed_width, static_cast<u32>(b->pages),
                       reinterpret_cast<u32*>(w + room.free_part), reinterpret_cast<u32*>(w + room.asked_part),
                       reinterpret_cast<u32*>(w + room.claim_part),
                       reinterpret_cast<u32*>(w + room.free_all), reinterpret_cast<int*>(w + room.claims),
                       reinterpret_cast<int*>(w + room.last), reinterpret_cast<int*>(w + room.pool), w + room.state};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    bool ok;
    if (const u32 team = cluster_size(b->pages, entries, u64{b->seqs} * ((b->width + 32 * kDeep - 1) / (32 * kDeep)))) {
        ok = cluster(resize_cluster_kernel, team, a, s);
    } else {
        const u32 blocks = pass_blocks();
        // counts that are where they belong need not be there before others change
        ok = (b->refs_out == b->refs ? pass(resize_pass_kernel<5>, blocks, false, a, s)
                                     : pass(resize_pass_kernel<0>, blocks, false, a, s) &&
                                           pass(resize_pass_kernel<1>, blocks, true, a, s)) &&
             pass(resize_pass_kernel<2>, blocks, true, a, s) && pass(resize_pass_kernel<3>, blocks, true, a, s) &&
             pass(resize_pass_kernel<4>, blocks, true, a, s);
    }
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

extern "C" int hbfsim_kv_fork_v1(const hbfsim_kv_fork_batch_v1* b, void* stream)
{
    if (!b || b->struct_size != sizeof(*b) || b->version != HBFSIM_KV_V1_VERSION) return HBFSIM_INVALID_ARGUMENT;
    if (b->block_tokens != 16 && b->block_tokens != 32 && b->block_tokens != 64) return HBFSIM_UNSUPPORTED;
    if (b->seqs > kKvMaxSeqs || b->rows > kKvMaxSeqs || b->width > kKvMaxWidth || b->pages > 0x7fffffffull ||
        u64{b->width} * b->block_tokens > 0x7fffffffull || !table_fits(b->seqs, b->width) ||
        !table_fits(b->rows, b->width))
        return HBFSIM_INVALID_ARGUMENT;
    if (b->seqs == 0 && b->rows == 0 && b->refs_out == b->refs) return HBFSIM_OK;
    const u64 entries = u64{b->seqs} * b->width, made = u64{b->rows} * b->width;
    if ((b->pages && (!b->refs || !b->refs_out)) || (entries && !b->table) || (b->seqs && !b->lengths) ||
        (b->rows && (!b->parents || !b->lengths_out)) || (made && !b->table_out))
        return HBFSIM_INVALID_ARGUMENT;
    for (const void* p : {static_cast<const void*>(b->refs), static_cast<const void*>(b->table),
                          static_cast<const void*>(b->lengths), static_cast<const void*>(b->parents),
                          static_cast<const void*>(b->refs_out), static_cast<const void*>(b->table_out),
                          static_cast<const void*>(b->lengths_out)})
        if (!kv_aligned(p, 4)) return HBFSIM_INVALID_ARGUMENT;
    const KvExtent out[] = {{b->refs_out, b->pages * 4}, {b->table_out, made * 4}, {b->lengths_out, u64{b->rows} * 4}};
    const KvExtent in[] = {{b->refs, b->pages * 4},
                         {b->table, b->seqs, b->width, b->table_stride},
                         {b->lengths, u64{b->seqs} * 4},
                         {b->parents, u64{b->rows} * 4}};
    if (kv_would_race(out, in, {0, -1, -1})) return HBFSIM_INVALID_ARGUMENT;
    const ForkArgs a{b->refs, b->table, b->table_stride, b->lengths, b->parents, b->refs_out, b->table_out,
                     b->lengths_out, b->seqs, b->rows, b->width, b->block_tokens, static_cast<u32>(b->pages)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool apart = b->refs_out != b->refs;
    // counts that are where they belong need no pass of their own
    const u32 blocks = pass_blocks();
    const bool ok = apart ? pass(fork_pass_kernel<0>, blocks, false, a, s) &&
                                pass(fork_pass_kernel<1>, blocks, true, a, s)
                          : pass(fork_pass_kernel<2>, blocks, false, a, s);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

static int compact_check(const hbfsim_kv_compact_batch_v1* b)
{
    if (!b || b->struct_size != sizeof(*b) || b->version != HBFSIM_KV_V1_VERSION) return HBFSIM_INVALID_ARGUMENT;
    if (b->seqs > kKvMaxSeqs || b->width > kKvMaxWidth || b->pages > 0x7fffffffull ||
        !table_fits(b->seqs, b->width))
        return HBFSIM_INVALID_ARGUMENT;
    return HBFSIM_OK;
}

extern "C" uint64_t hbfsim_kv_compact_workspace_v1(const hbfsim_kv_compact_batch_v1* b)
{
    return compact_check(b) == HBFSIM_OK ? part_bytes() : 0;
}

extern "C" int hbfsim_kv_compact_v1(const hbfsim_kv_compact_batch_v1* b, void* stream)
{
    if (const int rc = compact_check(b)) return rc;
    const u64 entries = u64{b->seqs} * b->width, room = b->pages / 2;
    if (!b->live || (b->pages && (!b->refs || !b->refs_out || !b->where)) || (room && (!b->src || !b->dst)) ||
        (entries && (!b->table || !b->table_out)) || !b->workspace)
        return HBFSIM_INVALID_ARGUMENT;
    for (const void* p : {static_cast<const void*>(b->refs), static_cast<const void*>(b->table),
                          static_cast<const void*>(b->refs_out), static_cast<const void*>(b->table_out),
                          static_cast<const void*>(b->src), static_cast<const void*>(b->dst),
                          static_cast<const void*>(b->live), static_cast<const void*>(b->where)})
        if (!kv_aligned(p, 4)) return HBFSIM_INVALID_ARGUMENT;
    if (!kv_aligned(b->workspace, 16) || b->workspace_bytes < part_bytes()) return HBFSIM_INVALID_ARGUMENT;
    if (entries && b->table_out == b->table && b->table_out_stride != b->table_stride) return HBFSIM_INVALID_ARGUMENT;
    if (b->seqs > 1 && std::abs(b->table_out_stride) < static_cast<i64>(b->width)) return HBFSIM_INVALID_ARGUMENT;
    const KvExtent out[] = {{b->refs_out, b->pages * 4}, {b->table_out, b->seqs, b->width, b->table_out_stride},
                          {b->src, room * 4},          {b->dst, room * 4},
                          {b->live, 4},                {b->where, b->pages * 4},
                          {b->workspace, part_bytes()}};
    const KvExtent in[] = {{b->refs, b->pages * 4}, {b->table, b->seqs, b->width, b->table_stride}};
    if (kv_would_race(out, in, {0, 1, -1, -1, -1, -1, -1})) return HBFSIM_INVALID_ARGUMENT;
    CompactArgs a{b->refs, b->table, b->table_stride, b->refs_out, b->table_out, b->table_out_stride, b->src,
                  b->dst, b->live, b->where, b->seqs, b->width, static_cast<u32>(b->pages),
                  static_cast<u32*>(b->workspace)};
    if (b->table_stride == static_cast<i64>(b->width) && b->table_out_stride == static_cast<i64>(b->width)) {
        a.seqs = 1;  // rows side by side are one: narrow ones would each take a warp
        a.width = static_cast<u32>(entries);
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    bool ok;
    if (b->pages <= kCompactMost && entries <= kCompactMost) {
        ok = cluster(compact_small_kernel, 1, a, s);
    } else {
        const u32 blocks = pass_blocks();
        ok = pass(compact_pass_kernel<0>, blocks, false, a, s) && pass(compact_pass_kernel<1>, blocks, true, a, s) &&
             pass(compact_pass_kernel<2>, blocks, true, a, s);
    }
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

extern "C" int hbfsim_kv_copy_v1(const hbfsim_kv_cache_v1* from, const hbfsim_kv_cache_v1* to, const int32_t* src,
                                 const int32_t* dst, uint64_t count, void* stream)
{
    CopyArgs a{};
    if (const int rc = kv_check_cache(from, a.from)) return rc;
    if (const int rc = kv_check_cache(to, a.to)) return rc;
    if (a.from.heads != a.to.heads || a.from.dim != a.to.dim || a.from.block != a.to.block || count > 0x7fffffffull)
        return HBFSIM_INVALID_ARGUMENT;
    if (count == 0) return HBFSIM_OK;
    if (!src || !dst || !kv_aligned(src, 4) || !kv_aligned(dst, 4)) return HBFSIM_INVALID_ARGUMENT;
    a.src = src;
    a.dst = dst;
    a.page_bytes = 2ull * a.from.heads * a.from.block * a.from.dim;
    a.per_page = static_cast<u32>((a.page_bytes + kCopyPiece - 1) / kCopyPiece);
    // thread blocks of several moves where there would be more than 512 to an SM
    a.count = count;
    a.group = static_cast<u32>(std::min<u64>(kCopyGroup, count * a.per_page / (512ull * kv_sm_count()) + 1));
    a.groups = (count + a.group - 1) / a.group;
    const u32 blocks = static_cast<u32>(std::min<u64>(a.groups * a.per_page, 0x7fffffffull));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool ok = kv_launch(copy_kernel, dim3(blocks), kCopyThreads, s, 0, 1, false, a);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
