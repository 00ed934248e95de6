// kv_select.cu -- block lists by a cheap score (kv_v1.h).
//
// A group's score of a block is linear in the block's bounds once the
// queries are split by sign: sum_d up_d * hi_d + down_d * lo_d with
// up = sum_g max(qi, 0), down = sum_g min(qi, 0).  So a block costs two dot
// products of 16-bit by 8-bit whole numbers (dp2a) per group instead of one
// pass per query head, and 2 * head_dim bytes, 1/16 of its keys and values
// at 16 tokens a block.
//
// score_kernel streams the bounds and writes a 32-bit ordered key per
// (token, head, block); list_kernel, one CTA per (sequence, token, head),
// finds the key of the last block to list by radix selection and writes the
// list in block order.
#include "kv.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace hbfb {
namespace {

constexpr u32 kScoreThreads = 256, kScoreBlocks = 64;  // blocks per CTA
constexpr u32 kListThreads = 256;
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

__device__ __forceinline__ float query_at(const KvQuery& q, u32 seq, u32 token, u32 head, u32 d)
{
    const i64 at = static_cast<i64>(seq) * q.stride_seq + static_cast<i64>(token) * q.stride_token +
                   static_cast<i64>(head) * q.stride_head + d;
    const float x = q.type == HBFSIM_KV_BF16
                        ? __bfloat162float(static_cast<const __nv_bfloat16*>(q.q)[at])
                        : __half2float(static_cast<const __half*>(q.q)[at]);
    return fabsf(x) <= 3.402823466e38f ? x : 0.0f;  // not finite: 0
}

// Blocks that a query token may look at: those up to its own position.
__device__ __forceinline__ u32 blocks_of_token(int length, u32 tokens, u32 t, u32 block)
{
    const int last = length - static_cast<int>(tokens) + static_cast<int>(t);
    return last < 0 ? 0u : static_cast<u32>(last) / block + 1u;
}

// Finite floats in their order, above kAbsent and below kAlways.
__device__ __forceinline__ u32 order_key(float x)
{
    const u32 b = __float_as_uint(fminf(x, 3.402823466e38f) + 0.0f);  // -0 becomes 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int D>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const SelectArgs a)
{
    constexpr u32 L = D / 16;   // lanes per (block, head): 16 channels each
    extern __shared__ __align__(16) short whole[];  // [tokens][heads][2][D]: up, down
    kv_let_next();
    const u32 seq = blockIdx.y, heads = a.c.heads, tokens = a.q.tokens, group = a.q.group;
    const int length = kv_length(a.q.lengths, seq, a.q.width, a.c.block);
    const u32 have = blocks_of_token(length, tokens, tokens - 1, a.c.block);
    const u32 first = blockIdx.x * kScoreBlocks;
    if (first >= have) return;
    const u32 many = min(kScoreBlocks, have - first);
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (u32 th = warp; th < tokens * heads; th += warps) {
        const u32 t = th / heads, h = th % heads;
        float most = 0.0f;
        for (u32 i = lane; i < group * D; i += 32)
            most = fmaxf(most, fabsf(query_at(a.q, seq, t, h * group + i / D, i % D)));
#pragma unroll
        for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        int x = 0;
        frexpf(most, &x);
        const float up_scale = kv_power(7 - max(x, -100));
        for (u32 d = lane; d < D; d += 32) {
            int up = 0, down = 0;
            for (u32 g = 0; g < group; ++g) {
                const float r = rintf(query_at(a.q, seq, t, h * group + g, d) * up_scale);
                const int qi = static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
                up += max(qi, 0);
                down += min(qi, 0);
            }
            whole[(th * 2) * D + d] = static_cast<short>(up);
            whole[(th * 2 + 1) * D + d] = static_cast<short>(down);
        }
    }
    __syncthreads();
    const int* table = a.q.table + static_cast<i64>(seq) * a.q.table_stride;
    const u32 part = threadIdx.x % L;
    const u32 items = many * heads;
    // every lane of a warp takes the same number of turns (the sums below shuffle)
    for (u32 base = warp * (32 / L); base < items; base += warps * (32 / L)) {
        const u32 item = base + lane / L;
        const bool in = item < items;
        const u32 j = first + (in ? item / heads : 0), h = in ? item % heads : 0;
        const int page = in ? kv_page(table, j, a.c.pages) : -1;
        uint4 lo{}, hi{};
        float scale = 0.0f;
        if (page >= 0) {
            const u64 at = static_cast<u64>(page) * heads + h;
            const uint4* b = reinterpret_cast<const uint4*>(a.c.bounds + at * 2 * D);
            lo = b[part];
            hi = b[L + part];
            scale = a.c.scale[at * 2];
        }
        for (u32 t = 0; t < tokens; ++t) {
            const int4* w = reinterpret_cast<const int4*>(whole + ((t * heads + h) * 2) * D + part * 16);
            const int4 u0 = w[0], u1 = w[1], n0 = w[D / 8], n1 = w[D / 8 + 1];
            int sum = 0;
            sum = __dp2a_lo(u0.x, static_cast<int>(hi.x), sum);
            sum = __dp2a_hi(u0.y, static_cast<int>(hi.x), sum);
            sum = __dp2a_lo(u0.z, static_cast<int>(hi.y), sum);
            sum = __dp2a_hi(u0.w, static_cast<int>(hi.y), sum);
            sum = __dp2a_lo(u1.x, static_cast<int>(hi.z), sum);
            sum = __dp2a_hi(u1.y, static_cast<int>(hi.z), sum);
            sum = __dp2a_lo(u1.z, static_cast<int>(hi.w), sum);
            sum = __dp2a_hi(u1.w, static_cast<int>(hi.w), sum);
            sum = __dp2a_lo(n0.x, static_cast<int>(lo.x), sum);
            sum = __dp2a_hi(n0.y, static_cast<int>(lo.x), sum);
            sum = __dp2a_lo(n0.z, static_cast<int>(lo.y), sum);
            sum = __dp2a_hi(n0.w, static_cast<int>(lo.y), sum);
            sum = __dp2a_lo(n1.x, static_cast<int>(lo.z), sum);
            sum = __dp2a_hi(n1.y, static_cast<int>(lo.z), sum);
            sum = __dp2a_lo(n1.z, static_cast<int>(lo.w), sum);
            sum = __dp2a_hi(n1.w, static_cast<int>(lo.w), sum);
#pragma unroll
            for (u32 o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (in && part == 0) {
                const u32 mine = blocks_of_token(length, tokens, t, a.c.block);
                u32 key = kAbsent;
                if (page >= 0 && j < mine) {
                    key = j < a.sink || j + a.recent >= mine
                              ? kAlways
                              : order_key(__fmul_rn(__int2float_rn(sum), scale));
                }
                a.keys[((static_cast<u64>(seq) * tokens + t) * heads + h) * a.q.width + j] = key;
            }
        }
    }
}

__global__ void __launch_bounds__(kListThreads) list_kernel(const SelectArgs a)
{
    __shared__ u32 histogram[256];
    __shared__ u32 shared2[2];
    __shared__ u32 warp_sums[33];
    kv_wait_before();
    const u64 at = blockIdx.x;  // (sequence, token, head)
    const u32 heads = a.c.heads, tokens = a.q.tokens;
    const u32 t = static_cast<u32>(at / heads % tokens), seq = static_cast<u32>(at / heads / tokens);
    const int length = kv_length(a.q.lengths, seq, a.q.width, a.c.block);
    const u32 have = blocks_of_token(length, tokens, t, a.c.block);
    const u32* keys = a.keys + at * a.q.width;
    int* list = a.blocks + at * a.top;
    // blocks that are there
    u32 mine = 0;
    for (u32 j = threadIdx.x; j < have; j += blockDim.x) mine += keys[j] != kAbsent;
    kv_block_scan(mine, warp_sums);
    const u32 present = warp_sums[32];
    const u32 take = min(a.top, present);
    // the greatest keys are the smallest of their complements
    u32 limit = 0xffffffffu, equals = 0;
    __syncthreads();
    if (take < present && take) {
        u32 below;
        limit = kv_select_rank<u32>(
            have, take,
            [&](u32 j, u32& k) {
                k = keys[j];
                if (k == kAbsent) return false;
                k = ~k;
                return true;
            },
            histogram, shared2, below);
        equals = take - below;
    }
    u32 listed_before = 0, equal_before = 0;
    for (u32 base = 0; base < have; base += blockDim.x) {
        const u32 j = base + threadIdx.x;
        const u32 key = j < have ? keys[j] : kAbsent;
        const bool in = key != kAbsent;
        bool listed = in;
        if (take < present) {
            const u32 equal = in && ~key == limit ? 1u : 0u;
            const u32 upto = equal_before + kv_block_scan(equal, warp_sums);
            equal_before += warp_sums[32];
            listed = in && (~key < limit || (equal && upto <= equals));
        }
        const u32 upto = listed_before + kv_block_scan(listed ? 1u : 0u, warp_sums);
        listed_before += warp_sums[32];
        if (listed && upto <= a.top) list[upto - 1] = static_cast<int>(j);
    }
    for (u32 i = take + threadIdx.x; i < a.top; i += blockDim.x) list[i] = -1;
    if (threadIdx.x == 0) a.counts[at] = static_cast<int>(take);
}

u64 workspace_bytes_of(const KvView& v, const KvQuery& q)
{
    return kv_round_up(static_cast<u64>(q.seqs) * q.tokens * v.heads * q.width * 4, 256);
}

template <int D>
int launch(const SelectArgs& a, cudaStream_t s)
{
    const u32 smem = a.q.tokens * a.c.heads * 2 * D * static_cast<u32>(sizeof(short));
    static std::atomic<u64> seen{0};
    if (!kv_allow_smem(score_kernel<D>, kMostQueryBytes, seen)) return HBFSIM_CUDA_ERROR;
    const dim3 grid((a.q.width + kScoreBlocks - 1) / kScoreBlocks, a.q.seqs);
    if (a.q.width) score_kernel<D><<<grid, kScoreThreads, smem, s>>>(a);
    const bool ok = kv_launch_behind(list_kernel, dim3(a.q.seqs * a.q.tokens * a.c.heads),
                                     kListThreads, s, a);
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
    if (static_cast<u64>(a.q.tokens) * a.c.heads * a.c.dim * 4 > kMostQueryBytes)
        return HBFSIM_UNSUPPORTED;
    if (a.q.seqs > 65535 || !blocks || !counts) return HBFSIM_INVALID_ARGUMENT;
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
