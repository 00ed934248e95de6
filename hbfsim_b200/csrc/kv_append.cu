// kv_append.cu -- new tokens into the 8-bit paged cache (kv_v1.h).
//
// One warp per (touched block, head, side).  A CTA's warps look at a chunk of
// up to 32 tokens, one per lane, and do the blocks whose first new token is
// among them, each warp for its head and side; few tokens get chunks of one,
// so that every block has a warp of its own at once.  A lane holds its
// channels of 16 tokens in registers between the two passes: the largest
// magnitude, which gives the scale, then the stored values (blocks of more
// tokens are read again).  Everything is a power of two away from the input,
// so the only rounding is the one to e4m3.
#include "kv.h"

#include <cuda_fp8.h>

#include <algorithm>

namespace hbfb {
namespace {

constexpr int kLowest = -100, kHighest = 120;

constexpr u32 kAppendWarps = 4;

struct AppendArgs {
    KvView c;
    const void* x[2];
    i64 stride_token[2], stride_head[2];
    bool wide[2];  // every head begins on a 16-byte boundary
    const int* table;
    i64 table_stride;
    const int* start;
    const int* offsets;
    u32 seqs, width, tokens, chunk;
};

// Two neighbouring elements of the input.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ u32 largest(u32 a, u32 b)  // of magnitudes; NaN loses
    {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const u32*>(&m);
    }
    static __device__ __forceinline__ float2 floats(u32 x)
    {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
};
template <>
struct Pair<__half> {
    static __device__ __forceinline__ u32 largest(u32 a, u32 b)
    {
        const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const u32*>(&m);
    }
    static __device__ __forceinline__ float2 floats(u32 x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
};

// Least e with a <= 448 * 2^e: a = m * 2^x, 0.5 <= m < 1, and 448 = 0.875 * 2^9.
__device__ __forceinline__ int scale_exponent(float a)
{
    if (!(a > 0.0f)) return kLowest;
    int x;
    const float m = frexpf(a, &x);
    return min(max(x - 9 + (m > 0.875f ? 1 : 0), kLowest), kHighest);
}

__device__ __forceinline__ float finite_or_0(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.0f; }

// N words of two stored values each, as f16 (exact).
__device__ __forceinline__ __half2 stored_f16(u32 two)
{
    return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3));
}

__device__ __forceinline__ u32 store_e4m3(float2 x)
{
    return __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
}

// A lane's channels of the new tokens among 16 rows of a block; 0 in the other rows.
template <int W>
__device__ __forceinline__ void load_rows(const u16* x, i64 stride, u32 row0, u32 slot, u32 count, bool wide,
                                          u32 (&raw)[16][W])
{
#pragma unroll
    for (u32 r = 0; r < 16; ++r) {
#pragma unroll
        for (int w = 0; w < W; ++w) raw[r][w] = 0;
        const u32 t = row0 + r - slot;  // wraps for earlier rows
        if (t < count) {
            const u16* from = x + t * stride;
            if (wide) {
                if constexpr (W == 1) {
                    raw[r][0] = *reinterpret_cast<const u32*>(from);
                } else if constexpr (W == 2) {
                    const uint2 y = *reinterpret_cast<const uint2*>(from);
                    raw[r][0] = y.x;
                    raw[r][1] = y.y;
                } else {
                    const uint4 y = *reinterpret_cast<const uint4*>(from);
                    raw[r][0] = y.x;
                    raw[r][1] = y.y;
                    raw[r][2] = y.z;
                    raw[r][3] = y.w;
                }
            } else {
#pragma unroll
                for (int w = 0; w < W; ++w) raw[r][w] = from[2 * w] | static_cast<u32>(from[2 * w + 1]) << 16;
            }
        }
    }
}

// One block, head and side by one warp.
template <typename T, int D>
__device__ __forceinline__ void append_block(const AppendArgs& a, u32 head, u32 side, u32 token, int page, u32 slot,
                                             u32 count)
{
    constexpr int W = D / 64;  // pairs of channels of a lane
    const u32 lane = threadIdx.x & 31u, block = a.c.block;
    const i64 stride = a.stride_token[side];
    const u16* x = static_cast<const u16*>(a.x[side]) + static_cast<i64>(token) * stride +
                   static_cast<i64>(head) * a.stride_head[side] + lane * 2 * W;
    const u64 at = (static_cast<u64>(page) * a.c.heads + head) * 2 + side;
    u8* out = a.c.data + at * block * D + lane * 2 * W;
    const float was = slot ? a.c.scale[at] : 0.0f;
    u32 raw[16][W];
    float most = 0.0f;
    for (u32 row0 = 0; row0 < block; row0 += 16) {
        if (row0 >= slot + count || row0 + 16 <= slot) continue;
        load_rows<W>(x, stride, row0, slot, count, a.wide[side], raw);
        u32 m = 0;
#pragma unroll
        for (u32 r = 0; r < 16; ++r)
#pragma unroll
            for (int w = 0; w < W; ++w) m = Pair<T>::largest(m, raw[r][w] & 0x7fff7fffu);
        float2 y = Pair<T>::floats(m);
        if (!(fmaxf(y.x, y.y) <= 3.402823466e38f)) {  // infinities: what is finite counts
            y = make_float2(0.0f, 0.0f);
#pragma unroll
            for (u32 r = 0; r < 16; ++r)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float2 z = Pair<T>::floats(raw[r][w]);
                    y.x = fmaxf(y.x, fmaxf(finite_or_0(z.x), finite_or_0(z.y)));
                }
        }
        most = fmaxf(most, fmaxf(y.x, y.y));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    float now = kv_power(scale_exponent(most));
    if (slot) now = fmaxf(now, was);
    __syncwarp();
    if (lane == 0) a.c.scale[at] = now;
    const float inverse = 1.0f / now, shrink = slot ? was / now : 1.0f;
    __half2 least[W], greatest[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        least[w] = __float2half2_rn(448.0f);
        greatest[w] = __float2half2_rn(-448.0f);
    }
    for (u32 row0 = 0; row0 < block; row0 += 16) {
        if (block > 16 && row0 < slot + count && row0 + 16 > slot)
            load_rows<W>(x, stride, row0, slot, count, a.wide[side], raw);
#pragma unroll
        for (u32 r = 0; r < 16; ++r) {
            const u32 row = row0 + r;
            u32 b[W];  // pairs of stored values
            bool write = true;
            if (row < slot) {
                write = shrink != 1.0f;
                if (!write && side) continue;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    b[w] = *reinterpret_cast<const u16*>(out + row * D + 2 * w);
                    if (write) {
                        float2 y = __half22float2(stored_f16(b[w]));
                        y.x *= shrink;
                        y.y *= shrink;
                        b[w] = store_e4m3(y);
                    }
                }
            } else if (row < slot + count) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    float2 y = Pair<T>::floats(raw[r][w]);
                    y.x *= inverse;
                    y.y *= inverse;
                    b[w] = store_e4m3(y);
                }
            } else {
#pragma unroll
                for (int w = 0; w < W; ++w) b[w] = 0;
            }
            if (write) {
                u8* to = out + row * D;
                if constexpr (W == 1) {
                    *reinterpret_cast<u16*>(to) = static_cast<u16>(b[0]);
                } else if constexpr (W == 2) {
                    *reinterpret_cast<u32*>(to) = b[0] | b[1] << 16;
                } else {
                    *reinterpret_cast<uint2*>(to) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
                }
            }
            if (side == 0 && row < slot + count) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    __half2 y = stored_f16(b[w]);
                    // NaN counts as 0
                    const u32 z = *reinterpret_cast<u32*>(&y) & __heq2_mask(y, y);
                    y = *reinterpret_cast<const __half2*>(&z);
                    least[w] = __hmin2(least[w], y);
                    greatest[w] = __hmax2(greatest[w], y);
                }
            }
        }
    }
    if (side == 0) {
        std::int8_t* bound = a.c.bounds + (static_cast<u64>(page) * a.c.heads + head) * 2 * D + lane * 2 * W;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 lo = __half22float2(least[w]), hi = __half22float2(greatest[w]);
            *reinterpret_cast<char2*>(bound + 2 * w) =
                make_char2(static_cast<signed char>(floorf(lo.x * 0.25f)), static_cast<signed char>(floorf(lo.y * 0.25f)));
            *reinterpret_cast<char2*>(bound + D + 2 * w) =
                make_char2(static_cast<signed char>(ceilf(hi.x * 0.25f)), static_cast<signed char>(ceilf(hi.y * 0.25f)));
        }
    }
}

// The last sequence that starts at or before a token, by a warp: 32 places at a time.
__device__ __forceinline__ u32 sequence_of(const AppendArgs& a, i64 token)
{
    const u32 lane = threadIdx.x & 31u;
    u32 lo = 0, hi = a.seqs;  // it is in [lo, hi)
    while (hi - lo > 1) {
        const u32 step = (hi - lo + 31) / 32, at = lo + lane * step;
        const u32 before = __ballot_sync(0xffffffffu, at < hi && (lane == 0 || a.offsets[at] <= token));
        const u32 last = 31 - __clz(before);  // offsets ascend: the lanes before it say yes as well
        hi = min(hi, lo + (last + 1) * step);
        lo += last * step;
    }
    return lo;
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(const AppendArgs a)
{
    const u32 lane = threadIdx.x & 31u;
    const u32 pair = blockIdx.y * kAppendWarps + (threadIdx.x >> 5), head = pair >> 1, side = pair & 1u;
    if (head >= a.c.heads) return;
    // the lane's token: its sequence, and whether it is the first new one of its block
    const i64 token = static_cast<i64>(blockIdx.x) * a.chunk + lane;
    bool leads = lane < a.chunk && token < a.tokens;
    int page = -1;
    u32 slot = 0, count = 0, seq_first = 0, seq_last = 0;
    if (a.offsets) {  // sequences of the chunk's first and last token
        const i64 base = static_cast<i64>(blockIdx.x) * a.chunk;
        seq_first = sequence_of(a, base);
        seq_last = a.chunk > 1 ? sequence_of(a, min(base + a.chunk, static_cast<i64>(a.tokens)) - 1) : seq_first;
    }
    if (leads) {
        u32 seq;
        i64 first, end;
        if (a.offsets) {
            u32 lo = seq_first, hi = seq_last + 1;  // offsets[lo] <= token < offsets[hi]
            leads = token >= a.offsets[0] && token < a.offsets[a.seqs];
            while (hi - lo > 1) {
                const u32 mid = (lo + hi) >> 1;
                if (token >= a.offsets[mid]) lo = mid;
                else hi = mid;
            }
            seq = lo;
            first = a.offsets[seq];
            end = min(static_cast<i64>(a.offsets[seq + 1]), static_cast<i64>(a.tokens));
        } else {
            const u32 each = a.tokens / a.seqs;
            seq = static_cast<u32>(token) / each;
            first = static_cast<i64>(seq) * each;
            end = first + each;
        }
        const i64 start = a.start[seq], position = start + (token - first);
        const u32 block = a.c.block;
        slot = static_cast<u32>(position) & (block - 1);
        const u64 j = static_cast<u64>(position) / block;
        leads = leads && start >= 0 && (slot == 0 || token == first) && j < a.width;
        if (leads) {
            page = kv_page(a.table + static_cast<i64>(seq) * a.table_stride, static_cast<u32>(j), a.c.pages);
            count = static_cast<u32>(min(static_cast<i64>(block - slot), end - token));
        }
        leads = leads && page >= 0;
    }
    for (u32 left = __ballot_sync(0xffffffffu, leads); left; left &= left - 1) {
        const int who = __ffs(left) - 1;
        append_block<T, D>(a, head, side, static_cast<u32>(blockIdx.x * a.chunk + who),
                           __shfl_sync(0xffffffffu, page, who), __shfl_sync(0xffffffffu, slot, who),
                           __shfl_sync(0xffffffffu, count, who));
    }
}

template <typename T>
int launch(const AppendArgs& a, cudaStream_t s)
{
    const dim3 grid((a.tokens + a.chunk - 1) / a.chunk, (a.c.heads * 2 + kAppendWarps - 1) / kAppendWarps);
    if (a.c.dim == 64) append_kernel<T, 64><<<grid, kAppendWarps * 32, 0, s>>>(a);
    else if (a.c.dim == 128) append_kernel<T, 128><<<grid, kAppendWarps * 32, 0, s>>>(a);
    else append_kernel<T, 256><<<grid, kAppendWarps * 32, 0, s>>>(a);
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
    auto wide = [](const void* p, i64 token, i64 head) { return kv_aligned(p, 16) && token % 8 == 0 && head % 8 == 0; };
    a.wide[0] = wide(b->k, b->k_stride_token, b->k_stride_head);
    a.wide[1] = wide(b->v, b->v_stride_token, b->v_stride_head);
    // one token to a chunk while all chunks' warps are resident at once (16 to an SM), more beyond
    a.chunk = 1;
    while (a.chunk < 32 && static_cast<u64>(a.tokens) * v.heads * 2 > static_cast<u64>(a.chunk) * 16 * kv_sm_count())
        a.chunk *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return b->type == HBFSIM_KV_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
}
