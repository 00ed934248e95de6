// kv.h -- shared pieces of the operators over the 8-bit paged key/value cache
// (include/hbfsim/kv_v1.h): argument checks, the device view of a cache, and
// the block-wide selection used by the block lists and the eviction.
#pragma once

#include "../../include/hbfsim/api.h"
#include "../../include/hbfsim/kv_v1.h"
#include "common.h"

#include <cuda_runtime.h>

#include <atomic>

namespace hbfb {

constexpr u32 kKvMaxTokens = 16;      // query tokens per sequence and call
constexpr u32 kKvMaxGroup = 64;       // query heads per key/value head
constexpr u32 kKvMaxWidth = 1u << 24; // blocks per sequence
constexpr u32 kKvMaxSeqs = 1u << 16;
constexpr u32 kKvMaxHeads = 1u << 10;

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
                  q->q_heads / v.heads, q->width, q->type};
    return HBFSIM_OK;
}

#if defined(__CUDACC__)
// Dynamic shared memory beyond 48 KB has to be allowed once per kernel and
// device; `seen` (one per kernel) remembers the devices.
template <typename Kernel>
inline bool kv_allow_smem(Kernel* kernel, u32 bytes, std::atomic<u64>& seen)
{
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return false;
    const u64 bit = device < 64 ? u64{1} << device : 0;
    if (seen.load(std::memory_order_acquire) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes)) != cudaSuccess)
        return false;
    seen.fetch_or(bit, std::memory_order_release);
    return true;
}

// Launches a kernel that may be set up while the kernel before it on the
// stream still runs (programmatic dependent launch): it has to begin with
// kv_wait_before, which returns once that kernel's writes are visible.
template <typename... Params, typename... Args>
inline bool kv_launch_behind(void (*kernel)(Params...), dim3 grid, u32 threads, cudaStream_t stream,
                             Args... args)
{
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...) == cudaSuccess;
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

// The `rank`-th smallest (from 1) of the keys key(0..n-1) that are not
// skipped, by 8-bit digits from the top: `histogram` (256 words) counts the
// digit among the keys that share the prefix found so far.  All threads call
// it; `below` gets how many keys are smaller than the result.
template <typename Key, typename KeyAt>
__device__ Key kv_select_rank(u32 n, u32 rank, KeyAt key_at, u32* histogram, u32* shared2,
                              u32& below)
{
    constexpr int kBits = sizeof(Key) * 8;
    Key prefix = 0;
    u32 left = rank;
    below = 0;
    for (int shift = kBits - 8; shift >= 0; shift -= 8) {
        for (u32 i = threadIdx.x; i < 256; i += blockDim.x) histogram[i] = 0;
        __syncthreads();
        for (u32 i = threadIdx.x; i < n; i += blockDim.x) {
            Key k;
            if (!key_at(i, k)) continue;
            if (shift + 8 < kBits && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
            atomicAdd(&histogram[static_cast<u32>(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x < 32) {  // one warp walks the 256 counts, 8 per lane
            u32 c[8], sum = 0;
#pragma unroll
            for (u32 t = 0; t < 8; ++t) {
                c[t] = histogram[threadIdx.x * 8 + t];
                sum += c[t];
            }
            u32 upto = sum;
#pragma unroll
            for (u32 o = 1; o < 32; o <<= 1) {
                const u32 y = __shfl_up_sync(0xffffffffu, upto, o);
                if (threadIdx.x >= o) upto += y;
            }
            u32 before = upto - sum;
            if (before < left && left <= upto) {
#pragma unroll
                for (u32 t = 0; t < 8; ++t) {
                    if (before < left && left <= before + c[t]) {
                        shared2[0] = threadIdx.x * 8 + t;
                        shared2[1] = before;
                    }
                    before += c[t];
                }
            }
        }
        __syncthreads();
        prefix |= static_cast<Key>(shared2[0]) << shift;
        left -= shared2[1];
        below += shared2[1];
        __syncthreads();
    }
    return prefix;
}

#endif  // __CUDACC__

}  // namespace hbfb
