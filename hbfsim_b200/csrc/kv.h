// kv.h -- shared pieces of the operators over the 8-bit paged key/value cache
// (include/hbfsim/kv_v1.h): argument checks, the device view of a cache, and
// the block-wide selection used by the block lists and the eviction.
#pragma once

#include "../../include/hbfsim/api.h"
#include "../../include/hbfsim/kv_v1.h"
#include "common.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

namespace hbfb {

constexpr u32 kKvMaxTokens = 16;      // query tokens per sequence and call
constexpr u32 kKvMaxGroup = 64;       // query heads per key/value head
constexpr u32 kKvMaxWidth = 1u << 24; // blocks per sequence
constexpr u32 kKvMaxSeqs = 1u << 16;
constexpr u32 kKvMaxHeads = 1u << 10;
constexpr u32 kKvTeam = 8;            // CTAs that select from one row at most

struct KvView {
    u8* data;
    float* scale;
    std::int8_t* bounds;
    u32 pages, heads, dim, block;
};

struct KvQuery {
    const void* q;
    i64 stride_seq, stride_token, stride_head;
    const int* table;
    i64 table_stride;
    const int* lengths;
    u32 seqs, tokens, q_heads, group, width, type;
    bool wide;  // every head begins on a 16-byte boundary
};

inline bool kv_aligned(const void* p, std::uintptr_t a)
{
    return reinterpret_cast<std::uintptr_t>(p) % a == 0;
}

// Checks a cache description; fills `v`.
inline int kv_check_cache(const hbfsim_kv_cache_v1* c, KvView& v)
{
    if (!c || c->struct_size != sizeof(*c) || c->version != HBFSIM_KV_V1_VERSION || c->reserved)
        return HBFSIM_INVALID_ARGUMENT;
    if (c->kv_heads == 0 || c->kv_heads > kKvMaxHeads || c->pages > 0x7fffffffull)
        return HBFSIM_INVALID_ARGUMENT;
    if ((c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) ||
        (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64))
        return HBFSIM_UNSUPPORTED;
    if (c->pages && (!c->data || !c->scale || !c->bounds)) return HBFSIM_INVALID_ARGUMENT;
    if (!kv_aligned(c->data, 16) || !kv_aligned(c->bounds, 16) || !kv_aligned(c->scale, 8))
        return HBFSIM_INVALID_ARGUMENT;
    v.data = static_cast<u8*>(c->data);
    v.scale = c->scale;
    v.bounds = c->bounds;
    v.pages = static_cast<u32>(c->pages);
    v.heads = c->kv_heads;
    v.dim = c->head_dim;
    v.block = c->block_tokens;
    return HBFSIM_OK;
}

inline int kv_check_query(const hbfsim_kv_query_v1* q, const KvView& v, KvQuery& out)
{
    if (!q || q->struct_size != sizeof(*q) || q->version != HBFSIM_KV_V1_VERSION || q->reserved)
        return HBFSIM_INVALID_ARGUMENT;
    if (q->type != HBFSIM_KV_BF16 && q->type != HBFSIM_KV_F16) return HBFSIM_UNSUPPORTED;
    if (q->tokens > kKvMaxTokens) return HBFSIM_UNSUPPORTED;
    if (q->q_heads == 0 || q->q_heads % v.heads || q->q_heads / v.heads > kKvMaxGroup ||
        q->seqs > kKvMaxSeqs || q->width > kKvMaxWidth)
        return HBFSIM_INVALID_ARGUMENT;
    if (static_cast<u64>(q->seqs) * q->tokens * q->q_heads > 0x7fffffffull ||
        static_cast<u64>(q->width) * v.block > 0x7fffffffull)
        return HBFSIM_INVALID_ARGUMENT;
    if (q->seqs && q->tokens) {
        if (!q->q || !q->lengths || (q->width && !q->table)) return HBFSIM_INVALID_ARGUMENT;
        if (!kv_aligned(q->q, 2) || !kv_aligned(q->table, 4) || !kv_aligned(q->lengths, 4))
            return HBFSIM_INVALID_ARGUMENT;
    }
    out = KvQuery{q->q, q->q_stride_seq, q->q_stride_token, q->q_stride_head, q->table,
                  q->table_stride, q->lengths, q->seqs, q->tokens, q->q_heads,
                  q->q_heads / v.heads, q->width, q->type,
                  kv_aligned(q->q, 16) && q->q_stride_seq % 8 == 0 &&
                      q->q_stride_token % 8 == 0 && q->q_stride_head % 8 == 0};
    return HBFSIM_OK;
}

// Whether a runtime call succeeded.  Calls report their own status and leave no error behind for
// the next one.
inline bool kv_ok(cudaError_t status)
{
    if (status != cudaSuccess) cudaGetLastError();
    return status == cudaSuccess;
}

inline int kv_sm_count()
{
    static std::atomic<int> counts[64];  // by device; the value does not change
    int device = 0;
    if (!kv_ok(cudaGetDevice(&device)) || device > 63) return 148;
    int n = counts[device].load(std::memory_order_relaxed);
    if (n == 0) {
        if (!kv_ok(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device)) || n <= 0) return 148;
        counts[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

#if defined(__CUDACC__)
// Dynamic shared memory beyond 48 KB has to be allowed once per kernel and
// device; `seen` (one per kernel) remembers the devices.
template <typename Kernel>
inline bool kv_allow_smem(Kernel* kernel, u32 bytes, std::atomic<u64>& seen)
{
    int device = 0;
    if (!kv_ok(cudaGetDevice(&device))) return false;
    const u64 bit = device < 64 ? u64{1} << device : 0;
    if (seen.load(std::memory_order_acquire) & bit) return true;
    if (!kv_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(bytes))))
        return false;
    seen.fetch_or(bit, std::memory_order_release);
    return true;
}

// CTAs to a row of `width` keys: a power of two up to kKvTeam, as long as
// every CTA gets an SM of its own and at least 2048 keys.
inline u32 kv_team_size(u64 rows, u32 width)
{
    u32 size = 1;
    while (size < kKvTeam && rows * size * 2 <= static_cast<u64>(kv_sm_count()) &&
           width / (size * 2) >= 2048)
        size *= 2;
    return size;
}

// Threads for a slice of a row: two keys each or more, a power of two (the
// bins are shared out evenly).
inline u32 kv_team_threads(u32 slice)
{
    return slice <= 256 ? 128 : slice <= 512 ? 256 : slice <= 1024 ? 512 : 1024;
}

// Launches a kernel in clusters of `cluster` CTAs.  `behind`: it may be set
// up while the kernel before it on the stream still runs (programmatic
// dependent launch); it then has to begin with kv_wait_before, which returns
// once that kernel's writes are visible.
template <typename... Params, typename... Args>
inline bool kv_launch(void (*kernel)(Params...), dim3 grid, u32 threads, cudaStream_t stream, u32 smem,
                      u32 cluster, bool behind, Args... args)
{
    cudaLaunchAttribute attributes[2]{};
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = attributes;
    if (behind) {
        attributes[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attributes[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attributes[config.numAttrs].val.clusterDim.x = cluster;
        attributes[config.numAttrs].val.clusterDim.y = 1;
        attributes[config.numAttrs++].val.clusterDim.z = 1;
    }
    return kv_ok(cudaLaunchKernelEx(&config, kernel, args...));
}

__device__ __forceinline__ void kv_wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void kv_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

inline u64 kv_round_up(u64 n, u64 to) { return (n + to - 1) / to * to; }

#if defined(__CUDACC__)

// Tokens of a sequence that the table can hold.
__device__ __forceinline__ int kv_length(const int* lengths, u32 seq, u32 width, u32 block)
{
    return min(max(lengths[seq], 0), static_cast<int>(width * block));
}

// Page of a block, or -1 for one that is not there.
__device__ __forceinline__ int kv_page(const int* table, u32 j, u32 pages)
{
    const int p = table[j];
    return static_cast<u32>(p) < pages ? p : -1;
}

// N neighbouring elements of a bf16 or f16 array from `at` on; `wide`: base
// and `at` allow loads of up to 16 bytes.
template <int N>
__device__ __forceinline__ void kv_load(const void* p, i64 at, u32 type, bool wide, float (&x)[N])
{
    const unsigned short* from = static_cast<const unsigned short*>(p) + at;
    u32 w[N / 2];  // pairs of elements
    if (wide) {
        if constexpr (N == 2) {
            w[0] = *reinterpret_cast<const u32*>(from);
        } else if constexpr (N == 4) {
            const uint2 y = *reinterpret_cast<const uint2*>(from);
            w[0] = y.x;
            w[1] = y.y;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 8) {
                const uint4 y = *reinterpret_cast<const uint4*>(from + i);
                w[i / 2] = y.x;
                w[i / 2 + 1] = y.y;
                w[i / 2 + 2] = y.z;
                w[i / 2 + 3] = y.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) w[i / 2] = from[i] | static_cast<u32>(from[i + 1]) << 16;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        if (type == HBFSIM_KV_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = y.x;
            x[2 * i + 1] = y.y;
        }
    }
}

// Asynchronous copies from global to shared memory.
__device__ __forceinline__ u32 kv_shared(const void* p) { return static_cast<u32>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void kv_copy16(u32 to, const void* from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void kv_copy16(void* to, const void* from) { kv_copy16(kv_shared(to), from); }
__device__ __forceinline__ void kv_copy8(u32 to, const void* from)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void kv_copy4(void* to, const void* from)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(kv_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void kv_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void kv_copy_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 2^e in 32 bits, -127 < e < 128.
__device__ __forceinline__ float kv_power(int e) { return __int_as_float((e + 127) << 23); }

// Inclusive scan over the block (up to 32 warps); `warp_sums` holds 33 words.
// Returns the inclusive prefix; total in warp_sums[32].
__device__ __forceinline__ u32 kv_block_scan(u32 x, u32* warp_sums)
{
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (u32 o = 1; o < 32; o <<= 1) {
        const u32 y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // earlier readers of warp_sums are done
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        u32 s = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
        for (u32 o = 1; o < 32; o <<= 1) {
            const u32 y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        if (lane < warps) warp_sums[lane] = s;
        if (lane == 31) warp_sums[32] = s;
    }
    __syncthreads();
    return x + (warp ? warp_sums[warp - 1] : 0);
}

// Selection over a row of keys by a team: one CTA, or a cluster of up to 8,
// each with a slice of the row, that count together through distributed
// shared memory (a row of 16,000 keys is bound by one SM's instructions).
constexpr u32 kKvBins = 2048, kKvWords = 1024;
struct KvSelectShared {
    u32 histogram[kKvBins];   // counts of the bins; also the prefix sums of `words`
    u32 group[kKvBins / 32];  // sums of 32 counts
    u32 words[kKvWords];
    u32 warp_sums[33];
    u32 found[3];             // bin, keys below it, keys in it
    u32 counts[2], in_front;
    u64 range[32][2], team_range[2];  // least and greatest key of the warps, of the CTA
    u32 tally[32][2], team_tally[2];  // the caller's two counts, likewise
    u64 few[32];              // the last candidates
    u32 few_count, few_equals;
    u64 few_limit;
};
constexpr u32 kKvAll = 0xffffffffu;

struct KvTeam {
    u32 rank, size;
};

__device__ __forceinline__ void kv_team_sync(const KvTeam& team)
{
    if (team.size == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// A word of the shared memory of another CTA of the team.
template <typename T>
__device__ __forceinline__ T kv_peek(const T* mine, u32 rank)
{
    u32 at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(at)
        : "r"(static_cast<u32>(__cvta_generic_to_shared(mine))), "r"(rank));
    T x;
    if constexpr (sizeof(T) == 8)
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(at) : "memory");
    else
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    return x;
}

// Sum of a word over the CTAs [0, ranks) of the team: one lane per CTA, all
// lanes of the warp get it.
__device__ __forceinline__ u32 kv_team_sum(const u32* mine, u32 ranks)
{
    const u32 lane = threadIdx.x & 31u;
    return __reduce_add_sync(0xffffffffu, lane < ranks ? kv_peek(mine, lane) : 0);
}

__device__ __forceinline__ int kv_top_bit(u32 x) { return 31 - __clz(static_cast<int>(x)); }
__device__ __forceinline__ int kv_top_bit(u64 x) { return 63 - __clzll(static_cast<long long>(x)); }

// What the team's threads found when they went over the keys: the least and
// greatest key (~0 and 0 without one) and two counts.  Clears the bins too.
template <typename Key>
__device__ void kv_gather(const KvTeam& team, KvSelectShared& sm, Key& least, Key& greatest, u32& tally0,
                          u32& tally1)
{
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    auto reduce = [&]() {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
            greatest = max(greatest, __shfl_xor_sync(0xffffffffu, greatest, o));
        }
        tally0 = __reduce_add_sync(0xffffffffu, tally0);
        tally1 = __reduce_add_sync(0xffffffffu, tally1);
    };
    reduce();
    if (lane == 0) {
        sm.range[warp][0] = least;
        sm.range[warp][1] = greatest;
        sm.tally[warp][0] = tally0;
        sm.tally[warp][1] = tally1;
    }
    for (u32 i = threadIdx.x; i < kKvBins; i += blockDim.x) sm.histogram[i] = 0;
    __syncthreads();
    const bool in = lane < blockDim.x >> 5;  // every warp for itself
    least = in ? static_cast<Key>(sm.range[lane][0]) : static_cast<Key>(~Key{0});
    greatest = in ? static_cast<Key>(sm.range[lane][1]) : Key{0};
    tally0 = in ? sm.tally[lane][0] : 0;
    tally1 = in ? sm.tally[lane][1] : 0;
    reduce();
    if (team.size == 1) return;
    if (threadIdx.x == 0) {
        sm.team_range[0] = least;
        sm.team_range[1] = greatest;
        sm.team_tally[0] = tally0;
        sm.team_tally[1] = tally1;
    }
    kv_team_sync(team);
    if (warp == 0) {  // one warp asks the other CTAs
        const bool ask = lane < team.size;
        least = ask ? static_cast<Key>(kv_peek(&sm.team_range[0], lane)) : static_cast<Key>(~Key{0});
        greatest = ask ? static_cast<Key>(kv_peek(&sm.team_range[1], lane)) : Key{0};
        tally0 = ask ? kv_peek(&sm.team_tally[0], lane) : 0;
        tally1 = ask ? kv_peek(&sm.team_tally[1], lane) : 0;
        reduce();
        if (lane == 0) {
            sm.range[0][0] = least;
            sm.range[0][1] = greatest;
            sm.tally[0][0] = tally0;
            sm.tally[0][1] = tally1;
        }
    }
    __syncthreads();
    least = static_cast<Key>(sm.range[0][0]);
    greatest = static_cast<Key>(sm.range[0][1]);
    tally0 = sm.tally[0][0];
    tally1 = sm.tally[0][1];
}

// Threshold of the `rank` smallest (rank >= 1) among the keys of the team
// that `key_at(i, k)` admits, i = 0..n-1 in each CTA, all in [lo, hi] (from
// kv_gather, which also cleared the bins): those below `limit` and `equals`
// of those at it (kKvAll: all of them).  Each pass spreads the keys of the
// range at hand over bins and goes on with the bin that holds the rank, until
// a warp can order what is in it.  The bins of the first pass grow with the
// distance from the least key (32 to an octave), so that sizes of many orders
// do not crowd a few counters; the 2048 of later passes are equal.  One pass
// is the rule for a few thousand keys; 64-bit keys take 7 at most.  All
// threads of the team call it.
template <typename Key, typename KeyAt>
__device__ void kv_rank_limit(const KvTeam& team, u32 n, u32 rank, Key lo, Key hi, KeyAt key_at,
                              KvSelectShared& sm, Key& limit, u32& equals)
{
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (bool octaves = true;; octaves = false) {
        if (lo >= hi) {  // one value is left
            limit = lo;
            equals = rank;
            return;
        }
        const int shift = max(0, kv_top_bit(static_cast<Key>(hi - lo)) + 1 - 11);
        auto octave_bin = [](Key d) -> u32 {
            if (d < 32) return static_cast<u32>(d);
            const int top = kv_top_bit(d);  // 5 bits below the top one
            return static_cast<u32>((top - 5) * 32) + static_cast<u32>(d >> (top - 5));
        };
        if (!octaves) {
            for (u32 i = threadIdx.x; i < kKvBins; i += blockDim.x) sm.histogram[i] = 0;
            __syncthreads();
        }
        if (threadIdx.x == 0) sm.few_count = 0;
        u32 at_lo = 0;  // keys at `lo` (blocks of no weight, say) would crowd one counter
        if (octaves) {
#pragma unroll 4
            for (u32 i = threadIdx.x; i < n; i += blockDim.x) {
                Key k;
                if (!key_at(i, k)) continue;
                if (k == lo) ++at_lo;
                else atomicAdd(&sm.histogram[octave_bin(static_cast<Key>(k - lo))], 1u);
            }
        } else {
            for (u32 i = threadIdx.x; i < n; i += blockDim.x) {
                Key k;
                if (!key_at(i, k) || k < lo || k > hi) continue;
                if (k == lo) ++at_lo;
                else atomicAdd(&sm.histogram[static_cast<u32>((k - lo) >> shift)], 1u);
            }
        }
        at_lo = __reduce_add_sync(0xffffffffu, at_lo);
        if (lane == 0 && at_lo) atomicAdd(&sm.histogram[0], at_lo);
        __syncthreads();
        if (team.size == 1) {
            const u32 each = kKvBins / blockDim.x, from = threadIdx.x * each;  // 2 to 16 bins a thread
            u32 sum = 0;
            for (u32 t = 0; t < each; ++t) sum += sm.histogram[from + t];
            u32 upto = sum;
#pragma unroll
            for (u32 o = 1; o < 32; o <<= 1) {
                const u32 y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            if (lane == 31) sm.warp_sums[warp] = upto;
            __syncthreads();
            upto += __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_sums[lane] : 0);
            u32 before = upto - sum;
            if (before < rank && rank <= upto) {
                u32 t = from;
                while (before + sm.histogram[t] < rank) before += sm.histogram[t++];
                sm.found[0] = t;
                sm.found[1] = before;
                sm.found[2] = sm.histogram[t];
            }
        } else {
            // Words of other CTAs are dear: first the sums of 32 bins each, then the 32 bins of
            // the group that holds the rank, by one warp.
            for (u32 w = warp; w < kKvBins / 32; w += warps) {
                const u32 sum = __reduce_add_sync(0xffffffffu, sm.histogram[w * 32 + lane]);
                if (lane == 0) sm.group[w] = sum;
            }
            kv_team_sync(team);
            if (warp == 0) {
                u32 before = 0, at = 0;
                // place of the rank among 32 counts, one per lane, each the team's sum
                auto narrow = [&](const u32* mine) -> bool {
                    u32 part[kKvTeam], sum = 0;  // all reads under way before the first sum
#pragma unroll
                    for (u32 r = 0; r < kKvTeam; ++r) part[r] = r < team.size ? kv_peek(mine + lane, r) : 0;
#pragma unroll
                    for (u32 r = 0; r < kKvTeam; ++r) sum += part[r];
                    u32 upto = sum;
#pragma unroll
                    for (u32 o = 1; o < 32; o <<= 1) {
                        const u32 y = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += y;
                    }
                    const u32 here = __ballot_sync(0xffffffffu, before + upto >= rank);
                    at = here ? __ffs(here) - 1 : 31;
                    const u32 in_front = __shfl_sync(0xffffffffu, upto - sum, at);
                    const u32 count = __shfl_sync(0xffffffffu, sum, at);
                    before += here ? in_front : __shfl_sync(0xffffffffu, upto, 31);
                    if (lane == 0) sm.found[2] = count;
                    return here != 0;
                };
                u32 group = 0;
                while (!narrow(sm.group + group) && group + 64 <= kKvBins / 32) group += 32;
                group += at;
                narrow(sm.histogram + group * 32);
                if (lane == 0) {
                    sm.found[0] = group * 32 + at;
                    sm.found[1] = before;
                }
            }
        }
        kv_team_sync(team);  // `found` is there, and nobody reads this CTA's counts any more
        const u32 bin = sm.found[0], count = sm.found[2];
        rank -= sm.found[1];
        int width = octaves ? 0 : shift;  // log2 of the bin's width
        if (octaves && bin >= 32) {
            width = static_cast<int>(bin / 32) - 1;
            lo += static_cast<Key>(32 + bin % 32) << width;
        } else {
            lo += static_cast<Key>(bin) << width;
        }
        const Key last = (Key{1} << width) - 1;  // lo + last may be past the type's range
        if (hi - lo > last) hi = lo + last;
        if (rank == count) {  // the whole bin
            limit = hi;
            equals = kKvAll;
            return;
        }
        if (count > 32) continue;
        // The bin's keys, one per lane, each ordered by how many are below it.
        for (u32 i = threadIdx.x; i < n; i += blockDim.x) {
            Key k;
            if (key_at(i, k) && k >= lo && k <= hi) sm.few[atomicAdd(&sm.few_count, 1u) & 31u] = k;
        }
        kv_team_sync(team);
        if (team.size == 1 || warp == 0) {  // every warp for itself, or one that asks the others
            Key k = static_cast<Key>(sm.few[lane]);
            if (team.size > 1) {
                u32 upto = 0;
                for (u32 r = 0; r < team.size; ++r) {
                    const u32 its = kv_peek(&sm.few_count, r);
                    if (lane >= upto && lane < upto + its) k = static_cast<Key>(kv_peek(&sm.few[lane - upto], r));
                    upto += its;
                }
            }
            u32 below = 0, same = 0;
            for (u32 x = 0; x < count; ++x) {
                const Key other = __shfl_sync(0xffffffffu, k, x);
                below += other < k;
                same += other == k;
            }
            const bool it = lane < count && below < rank && rank <= below + same;
            const u32 who = __ballot_sync(0xffffffffu, it);
            const int one = who ? __ffs(who) - 1 : 0;
            limit = __shfl_sync(0xffffffffu, k, one);
            equals = rank - __shfl_sync(0xffffffffu, below, one);
            if (equals == __shfl_sync(0xffffffffu, same, one)) equals = kKvAll;
            if (lane == 0 && team.size > 1) {
                sm.few_limit = limit;
                sm.few_equals = equals;
            }
        }
        if (team.size > 1) {
            __syncthreads();
            limit = static_cast<Key>(sm.few_limit);
            equals = sm.few_equals;
        }
        return;
    }
}

// Walks the team's elements in order (0..n-1 in each CTA, CTAs by rank; with
// more than one CTA n is at most 32768): state(i) is 0 (not chosen), 1
// (chosen) or 2 (one of the equals, of which the first `equals` are chosen).
// For every i, value = load(i), then store(i, value, chosen, how many chosen
// came before), with a block barrier between them if kBarrier (stores may
// reach what a load of the same round reads).  Counts come from ballots, one
// word per 32 elements, and one block-wide scan per 32768 elements.
template <bool kBarrier, bool kChosen, typename State, typename Load, typename Store>
__device__ void kv_walk(const KvTeam& team, u32 n, u32 equals, KvSelectShared& sm, State state,
                        Load load, Store store)
{
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const u32 under = (1u << lane) - 1u;
    u32* prefix = sm.histogram;
    u32 before[2] = {0, 0};  // chosen, equals in front of the elements at hand
    // Exclusive prefix sums of the words' bit counts; returns their sum.  A team's CTAs add
    // what the ones in front counted to before[which].
    auto scan_words = [&](u32 many, int which) {
        u32 carry = 0;
        if (many <= 128) {  // every warp for itself: they write the same
            for (u32 base = 0; base < many; base += 32) {
                const u32 w = base + lane, bits = w < many ? __popc(sm.words[w]) : 0;
                u32 upto = bits;
#pragma unroll
                for (u32 o = 1; o < 32; o <<= 1) {
                    const u32 y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                if (w < many) prefix[w] = carry + upto - bits;
                carry += __shfl_sync(0xffffffffu, upto, 31);
            }
            __syncwarp();
        } else {
            for (u32 base = 0; base < many; base += blockDim.x) {
                const u32 w = base + threadIdx.x;
                const u32 bits = w < many ? __popc(sm.words[w]) : 0;
                const u32 upto = kv_block_scan(bits, sm.warp_sums);
                if (w < many) prefix[w] = carry + upto - bits;
                carry += sm.warp_sums[32];
            }
            __syncthreads();
        }
        if (team.size > 1) {
            if (threadIdx.x == 0) sm.counts[which] = carry;
            kv_team_sync(team);
            if (warp == 0) {
                const u32 sum = kv_team_sum(&sm.counts[which], team.rank);
                if (lane == 0) sm.in_front = sum;
            }
            __syncthreads();
            before[which] += sm.in_front;
        }
        return carry;
    };
    u32 first = 0;
    do {
        const u32 many = min(n - first, kKvWords * 32), words = (many + 31) / 32;
        const u32 rounds = (words + warps - 1) / warps;
        __syncthreads();
        if (equals != kKvAll) {
            for (u32 r = 0; r < rounds; ++r) {
                const u32 w = r * warps + warp, i = w * 32 + lane;
                const u32 m = __ballot_sync(0xffffffffu, i < many && state(first + i) == 2);
                if (lane == 0 && w < words) sm.words[w] = m;
            }
            __syncthreads();
            const u32 all = scan_words(words, 1);
            __syncthreads();  // every warp has read the words
            // from here on they hold what is chosen; a warp reads and writes its own words
            for (u32 r = 0; r < rounds; ++r) {
                const u32 w = r * warps + warp, i = w * 32 + lane;
                const u32 eq = w < words ? sm.words[w] : 0;
                const bool one = i < many && state(first + i) == 1;
                const bool rank_ok = w < words && before[1] + prefix[w] + __popc(eq & under) < equals;
                const u32 m = __ballot_sync(0xffffffffu, one || ((eq >> lane & 1u) && rank_ok));
                if (lane == 0 && w < words) sm.words[w] = m;
            }
            before[1] += all;
        } else {
            for (u32 r = 0; r < rounds; ++r) {
                const u32 w = r * warps + warp, i = w * 32 + lane;
                const u32 m = __ballot_sync(0xffffffffu, i < many && state(first + i) != 0);
                if (lane == 0 && w < words) sm.words[w] = m;
            }
        }
        __syncthreads();
        // (the prefix sums in use above are read: a barrier lies behind)
        const u32 all = scan_words(words, 0);
        for (u32 r = 0; r < rounds; ++r) {
            const u32 w = r * warps + warp, i = w * 32 + lane;
            const bool in = i < many;
            if constexpr (kChosen && !kBarrier) {
                if (w >= words || sm.words[w] == 0) continue;  // a warp at once
            }
            auto value = load(first + (in ? i : 0));
            if constexpr (kBarrier) __syncthreads();
            if (in) {
                const u32 m = sm.words[w];
                const bool chosen = (m >> lane & 1u) != 0;
                if (!kChosen || chosen)
                    store(first + i, value, chosen, before[0] + prefix[w] + __popc(m & under));
            }
        }
        before[0] += all;
        first += kKvWords * 32;
    } while (first < n);
}

#endif  // __CUDACC__

}  // namespace hbfb
