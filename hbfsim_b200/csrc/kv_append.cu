// kv_append.cu -- new tokens into the 8-bit paged cache (kv_v1.h).
//
// One warp per (touched block, head, side).  A warp is launched for every
// (token, head, side); the one whose token is the first new one of its block
// does the block, the others leave.  Two passes over the block's new tokens
// (the second reads them from L1/L2): the largest magnitude, which gives the
// scale, then the stored values.  Everything is a power of two away from the
// input, so the only rounding is the one to e4m3.
#include "kv.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace hbfb {
namespace {

constexpr int kLowest = -100, kHighest = 120;

struct AppendArgs {
    KvView c;
    const void* x[2];
    i64 stride_token[2], stride_head[2];
    const int* table;
    i64 table_stride;
    const int* start;
    const int* offsets;
    u32 seqs, width, tokens;
};

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// Least e with a <= 448 * 2^e: a = m * 2^x, 0.5 <= m < 1, and 448 = 0.875 * 2^9.
__device__ __forceinline__ int scale_exponent(float a)
{
    if (!(a > 0.0f)) return kLowest;
    int x;
    const float m = frexpf(a, &x);
    return min(max(x - 9 + (m > 0.875f ? 1 : 0), kLowest), kHighest);
}

__device__ __forceinline__ float from_e4m3(u8 b)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

template <typename T, int D>
__global__ void __launch_bounds__(128) append_kernel(const AppendArgs a)
{
    constexpr int E = D / 32;  // channels per lane
    const u32 lane = threadIdx.x & 31u;
    const u64 item = (static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const u32 side = item & 1u;
    const u64 rest = item >> 1;
    const u32 head = static_cast<u32>(rest % a.c.heads);
    const u64 token = rest / a.c.heads;
    if (token >= a.tokens) return;
    // the token's sequence: the last one that starts at or before it
    u32 seq;
    i64 first, end;
    if (a.offsets) {
        u32 lo = 0, hi = a.seqs;  // offsets[lo] <= token < offsets[hi]
        if (static_cast<i64>(token) < a.offsets[0] || static_cast<i64>(token) >= a.offsets[hi])
            return;
        while (hi - lo > 1) {
            const u32 mid = (lo + hi) >> 1;
            if (static_cast<i64>(token) >= a.offsets[mid]) lo = mid;
            else hi = mid;
        }
        seq = lo;
        first = a.offsets[seq];
        end = min(static_cast<i64>(a.offsets[seq + 1]), static_cast<i64>(a.tokens));
    } else {
        const u32 each = a.tokens / a.seqs;
        seq = static_cast<u32>(token / each);
        first = static_cast<i64>(seq) * each;
        end = first + each;
    }
    const i64 start = a.start[seq];
    if (start < 0) return;
    const i64 position = start + (static_cast<i64>(token) - first);
    const u32 block = a.c.block;
    const u32 slot = static_cast<u32>(position % block);
    if (slot != 0 && static_cast<i64>(token) != first) return;  // not its block's first new token
    const i64 j = position / block;
    if (j >= a.width) return;
    const int page = kv_page(a.table + static_cast<i64>(seq) * a.table_stride, static_cast<u32>(j),
                             a.c.pages);
    if (page < 0) return;
    const u32 count = static_cast<u32>(min(static_cast<i64>(block - slot), end - static_cast<i64>(token)));
    const T* x = static_cast<const T*>(a.x[side]) + static_cast<i64>(token) * a.stride_token[side] +
                 static_cast<i64>(head) * a.stride_head[side] + lane * E;
    float most = 0.0f;
    for (u32 t = 0; t < count; ++t)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float v = fabsf(to_float(x[t * a.stride_token[side] + i]));
            if (v <= 3.402823466e38f) most = fmaxf(most, v);  // finite
        }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const u64 at = (static_cast<u64>(page) * a.c.heads + head) * 2 + side;
    float now = kv_power(scale_exponent(most));
    const float was = slot ? a.c.scale[at] : now;
    now = fmaxf(now, was);
    __syncwarp();
    if (lane == 0) a.c.scale[at] = now;
    const float inverse = 1.0f / now, shrink = was / now;
    u8* out = a.c.data + at * block * D + lane * E;
    float least[E], greatest[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        least[i] = 448.0f;
        greatest[i] = -448.0f;
    }
    for (u32 t = 0; t < block; ++t) {
        u8 b[E];
        if (t < slot) {
#pragma unroll
            for (int i = 0; i < E; ++i) b[i] = out[t * D + i];
            if (shrink != 1.0f) {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    b[i] = __nv_cvt_float_to_fp8(from_e4m3(b[i]) * shrink, __NV_SATFINITE, __NV_E4M3);
            }
        } else if (t < slot + count) {
#pragma unroll
            for (int i = 0; i < E; ++i)
                b[i] = __nv_cvt_float_to_fp8(
                    to_float(x[(t - slot) * a.stride_token[side] + i]) * inverse, __NV_SATFINITE,
                    __NV_E4M3);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) b[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) out[t * D + i] = b[i];
        if (side == 0 && t < slot + count) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                float v = from_e4m3(b[i]);
                v = v == v ? v : 0.0f;
                least[i] = fminf(least[i], v);
                greatest[i] = fmaxf(greatest[i], v);
            }
        }
    }
    if (side == 0) {
        std::int8_t* bound = a.c.bounds + (static_cast<u64>(page) * a.c.heads + head) * 2 * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            bound[i] = static_cast<std::int8_t>(floorf(least[i] * 0.25f));
            bound[D + i] = static_cast<std::int8_t>(ceilf(greatest[i] * 0.25f));
        }
    }
}

template <typename T>
int launch(const AppendArgs& a, cudaStream_t s)
{
    const u64 warps = static_cast<u64>(a.tokens) * a.c.heads * 2;
    const u32 grid = static_cast<u32>((warps + 3) / 4);
    if (a.c.dim == 64) append_kernel<T, 64><<<grid, 128, 0, s>>>(a);
    else if (a.c.dim == 128) append_kernel<T, 128><<<grid, 128, 0, s>>>(a);
    else append_kernel<T, 256><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" int hbfsim_kv_append_v1(const hbfsim_kv_cache_v1* cache,
                                   const hbfsim_kv_append_batch_v1* b, void* stream)
{
    KvView v{};
    if (const int rc = kv_check_cache(cache, v)) return rc;
    if (!b || b->struct_size != sizeof(*b) || b->version != HBFSIM_KV_V1_VERSION || b->reserved)
        return HBFSIM_INVALID_ARGUMENT;
    if (b->type != HBFSIM_KV_BF16 && b->type != HBFSIM_KV_F16) return HBFSIM_UNSUPPORTED;
    if (b->seqs > kKvMaxSeqs || b->width > kKvMaxWidth || b->tokens > (1u << 22))
        return HBFSIM_INVALID_ARGUMENT;
    if (b->tokens == 0) return HBFSIM_OK;
    if (b->seqs == 0 || (!b->offsets && b->tokens % b->seqs)) return HBFSIM_INVALID_ARGUMENT;
    if (!b->k || !b->v || !b->start || (b->width && !b->table)) return HBFSIM_INVALID_ARGUMENT;
    if (!kv_aligned(b->k, 2) || !kv_aligned(b->v, 2) || !kv_aligned(b->table, 4) ||
        !kv_aligned(b->start, 4) || !kv_aligned(b->offsets, 4))
        return HBFSIM_INVALID_ARGUMENT;
    if (b->width == 0 || v.pages == 0) return HBFSIM_OK;  // no block is there
    AppendArgs a{};
    a.c = v;
    a.x[0] = b->k;
    a.x[1] = b->v;
    a.stride_token[0] = b->k_stride_token;
    a.stride_token[1] = b->v_stride_token;
    a.stride_head[0] = b->k_stride_head;
    a.stride_head[1] = b->v_stride_head;
    a.table = b->table;
    a.table_stride = b->table_stride;
    a.start = b->start;
    a.offsets = b->offsets;
    a.seqs = b->seqs;
    a.width = b->width;
    a.tokens = static_cast<u32>(b->tokens);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return b->type == HBFSIM_KV_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
}
