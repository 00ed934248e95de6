// kv_append.cuh -- what the appends to the 8-bit paged cache share (kv_append.cu, kv_rotary.cu):
// rows of the input, stored values, the search for the blocks of a chunk of tokens, and a block of
// new keys or values by one warp.
#pragma once

#include "kv.h"

#include <cuda_fp8.h>

#include <type_traits>

namespace hbfb {
namespace {

constexpr int kLowest = -100, kHighest = 120;

struct AppendArgs {
    KvView c;
    const void* x[2];
    i64 stride_token[2], stride_head[2];
    bool wide;  // every head of k and v begins on a 16-byte boundary
    const int* table;
    i64 table_stride;
    const int* start;
    const int* offsets;
    u32 seqs, width, tokens, chunk;
};

// Whether every head's row begins on a 16-byte boundary.
inline bool kv_rows_wide(const void* p, i64 token, i64 head)
{
    return kv_aligned(p, 16) && token % 8 == 0 && head % 8 == 0;
}

// Checks the arguments of an append and fills `a` but for the chunk.
inline int append_check(const hbfsim_kv_cache_v1* cache, const hbfsim_kv_append_batch_v1* b, AppendArgs& a)
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
    a.wide = kv_rows_wide(b->k, b->k_stride_token, b->k_stride_head) &&
             kv_rows_wide(b->v, b->v_stride_token, b->v_stride_head);
    return HBFSIM_OK;
}

// Two neighbouring elements of the input.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
    // the lesser and the greater of each, NaN if either is
    static __device__ __forceinline__ void span(u32& lo, u32& hi, u32 x)
    {
        const __nv_bfloat162 y = *reinterpret_cast<__nv_bfloat162*>(&x);
        const __nv_bfloat162 l = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&lo), y);
        const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&hi), y);
        lo = *reinterpret_cast<const u32*>(&l);
        hi = *reinterpret_cast<const u32*>(&h);
    }
    static __device__ __forceinline__ float2 floats(u32 x)
    {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
};
template <>
struct Pair<__half> {
    static __device__ __forceinline__ void span(u32& lo, u32& hi, u32 x)
    {
        const __half2 y = *reinterpret_cast<__half2*>(&x);
        const __half2 l = __hmin2_nan(*reinterpret_cast<__half2*>(&lo), y);
        const __half2 h = __hmax2_nan(*reinterpret_cast<__half2*>(&hi), y);
        lo = *reinterpret_cast<const u32*>(&l);
        hi = *reinterpret_cast<const u32*>(&h);
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

// A lane's channels of one token.
template <int W, bool kWide>
__device__ __forceinline__ void load_row(const u16* from, u32 (&raw)[W])
{
    if constexpr (!kWide) {
#pragma unroll
        for (int w = 0; w < W; ++w) raw[w] = from[2 * w] | static_cast<u32>(from[2 * w + 1]) << 16;
    } else if constexpr (W == 1) {
        raw[0] = *reinterpret_cast<const u32*>(from);
    } else if constexpr (W == 2) {
        const uint2 y = *reinterpret_cast<const uint2*>(from);
        raw[0] = y.x;
        raw[1] = y.y;
    } else {
        const uint4 y = *reinterpret_cast<const uint4*>(from);
        raw[0] = y.x;
        raw[1] = y.y;
        raw[2] = y.z;
        raw[3] = y.w;
    }
}

// Bounds of a lane's channels from the least and greatest stored values (pairs).
template <int D>
__device__ __forceinline__ void put_bounds(const AppendArgs& a, int page, u32 head, const u32 (&lo)[D / 64],
                                           const u32 (&hi)[D / 64])
{
    constexpr int W = D / 64;
    std::int8_t* bound = a.c.bounds + (static_cast<u64>(page) * a.c.heads + head) * 2 * D + (threadIdx.x & 31u) * 2 * W;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float2 l = __half22float2(stored_f16(lo[w])), h = __half22float2(stored_f16(hi[w]));
        *reinterpret_cast<char2*>(bound + 2 * w) =
            make_char2(static_cast<signed char>(floorf(l.x * 0.25f)), static_cast<signed char>(floorf(l.y * 0.25f)));
        *reinterpret_cast<char2*>(bound + D + 2 * w) =
            make_char2(static_cast<signed char>(ceilf(h.x * 0.25f)), static_cast<signed char>(ceilf(h.y * 0.25f)));
    }
}

// A row's stored values.
template <int W>
__device__ __forceinline__ void put_row(u8* to, const u32 (&b)[W])
{
    if constexpr (W == 1) *reinterpret_cast<u16*>(to) = static_cast<u16>(b[0]);
    else if constexpr (W == 2) *reinterpret_cast<u32*>(to) = b[0] | b[1] << 16;
    else *reinterpret_cast<uint2*>(to) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
}

// A block whose tokens are all new, head and side by one warp; false, with
// nothing written, where an element is not finite.  Rounding keeps the order,
// so the least and greatest of the input give both the scale and the bounds.
template <typename T, int D, bool kWide>
__device__ __forceinline__ bool append_full(const AppendArgs& a, u32 head, u32 side, u32 token, int page)
{
    constexpr int W = D / 64;  // pairs of channels of a lane
    const u32 lane = threadIdx.x & 31u, block = a.c.block;
    const i64 stride = a.stride_token[side];
    const u16* x = static_cast<const u16*>(a.x[side]) + static_cast<i64>(token) * stride +
                   static_cast<i64>(head) * a.stride_head[side] + lane * 2 * W;
    const u64 at = (static_cast<u64>(page) * a.c.heads + head) * 2 + side;
    u32 raw[16][W], lo[W], hi[W];
    auto load_rows = [&](u32 row0) {
#pragma unroll
        for (u32 r = 0; r < 16; ++r) load_row<W, kWide>(x + (row0 + r) * stride, raw[r]);
    };
    load_rows(0);
#pragma unroll
    for (int w = 0; w < W; ++w) lo[w] = hi[w] = raw[0][w];
    for (u32 row0 = 0;;) {
#pragma unroll
        for (u32 r = 0; r < 16; ++r)
#pragma unroll
            for (int w = 0; w < W; ++w) Pair<T>::span(lo[w], hi[w], raw[r][w]);
        row0 += 16;
        if (row0 == block) break;
        load_rows(row0);
    }
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float2 l = Pair<T>::floats(lo[w]), h = Pair<T>::floats(hi[w]);
        const float m = fmaxf(fmaxf(fabsf(l.x), fabsf(l.y)), fmaxf(fabsf(h.x), fabsf(h.y)));
        finite &= m <= 3.402823466e38f && l.x == l.x && l.y == l.y;
        most = fmaxf(most, m);
    }
    if (!__all_sync(0xffffffffu, finite)) return false;
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float now = kv_power(scale_exponent(most)), inverse = 1.0f / now;
    if (lane == 0) a.c.scale[at] = now;
    auto stored = [&](u32 pair) {
        float2 y = Pair<T>::floats(pair);
        y.x *= inverse;
        y.y *= inverse;
        return store_e4m3(y);
    };
    u8* out = a.c.data + at * block * D + lane * 2 * W;
    for (u32 row0 = 0;;) {
        if (block > 16) load_rows(row0);
#pragma unroll
        for (u32 r = 0; r < 16; ++r) {
            u32 b[W];
#pragma unroll
            for (int w = 0; w < W; ++w) b[w] = stored(raw[r][w]);
            put_row<W>(out + (row0 + r) * D, b);
        }
        row0 += 16;
        if (row0 == block) break;
    }
    if (side == 0) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            lo[w] = stored(lo[w]);
            hi[w] = stored(hi[w]);
        }
        put_bounds<D>(a, page, head, lo, hi);
    }
    return true;
}

// Any block, head and side by one warp: `slot` tokens held before, `count` new ones, whose row(t, y)
// gives a lane's channels of token t in 32 bits.
template <int D, typename Row>
__device__ __forceinline__ void append_block(const AppendArgs& a, u32 head, u32 side, int page, u32 slot, u32 count,
                                             const Row& row)
{
    constexpr int W = D / 64;  // pairs of channels of a lane
    const u32 lane = threadIdx.x & 31u, block = a.c.block;
    const u64 at = (static_cast<u64>(page) * a.c.heads + head) * 2 + side;
    u8* out = a.c.data + at * block * D + lane * 2 * W;
    // what 16 rows hold, all reads under way at once
    constexpr int H = W == 4 ? 2 : 1;  // words of a lane's stored values in a row
    u32 held[16][H];
    auto load_held = [&](u32 row0) {
#pragma unroll
        for (u32 r = 0; r < 16; ++r) {
#pragma unroll
            for (int w = 0; w < H; ++w) held[r][w] = 0;
            if (row0 + r < slot) {
                const u8* from = out + (row0 + r) * D;
                if constexpr (W == 1) {
                    held[r][0] = *reinterpret_cast<const u16*>(from);
                } else {
#pragma unroll
                    for (int w = 0; w < H; ++w) held[r][w] = reinterpret_cast<const u32*>(from)[w];
                }
            }
        }
    };
    if (side == 0) load_held(0);  // the keys' bounds need them in any case
    const float was = slot ? a.c.scale[at] : 0.0f;
    float most = 0.0f;
#pragma unroll Row::kAhead
    for (u32 t = 0; t < count; ++t) {
        float2 y[W];
        row(t, y);
#pragma unroll
        for (int w = 0; w < W; ++w) most = fmaxf(most, fmaxf(finite_or_0(y[w].x), finite_or_0(y[w].y)));
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
    auto bound = [&](const u32 (&b)[W]) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            __half2 y = stored_f16(b[w]);
            // NaN counts as 0
            const u32 z = *reinterpret_cast<u32*>(&y) & __heq2_mask(y, y);
            y = *reinterpret_cast<const __half2*>(&z);
            least[w] = __hmin2(least[w], y);
            greatest[w] = __hmax2(greatest[w], y);
        }
    };
    if (side == 0 || shrink != 1.0f) {  // values need nothing else
        for (u32 row0 = 0; row0 < slot; row0 += 16) {
            if (row0 || side) load_held(row0);
#pragma unroll
            for (u32 r = 0; r < 16; ++r) {
                if (row0 + r >= slot) break;
                u32 b[W];
#pragma unroll
                for (int w = 0; w < W; ++w) b[w] = held[r][w / 2] >> (w & 1) * 16 & 0xffffu;
                if (shrink != 1.0f) {
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        float2 y = __half22float2(stored_f16(b[w]));
                        y.x *= shrink;
                        y.y *= shrink;
                        b[w] = store_e4m3(y);
                    }
                    put_row<W>(out + (row0 + r) * D, b);
                }
                if (side == 0) bound(b);
            }
        }
    }
#pragma unroll 2
    for (u32 t = 0; t < count; ++t) {
        float2 y[W];
        u32 b[W];
        row(t, y);
#pragma unroll
        for (int w = 0; w < W; ++w) b[w] = store_e4m3(make_float2(y[w].x * inverse, y[w].y * inverse));
        put_row<W>(out + (slot + t) * D, b);
        if (side == 0) bound(b);
    }
    const u32 none[W] = {};
    for (u32 r = slot + count; r < block; ++r) put_row<W>(out + r * D, none);
    if (side == 0) {
        u32 lo[W], hi[W];  // the values are stored ones: rounding them again changes nothing
#pragma unroll
        for (int w = 0; w < W; ++w) {
            lo[w] = store_e4m3(__half22float2(least[w]));
            hi[w] = store_e4m3(__half22float2(greatest[w]));
        }
        put_bounds<D>(a, page, head, lo, hi);
    }
}

// A head's new keys or values as they are: the `row` of append_block.  kAhead: rows that the search for the
// scale has under way.  Four instead of two take 38.4 instead of 41.8 us for 40 sequences of 200 tokens (256
// channels, blocks of 64), 4.95 instead of 5.15 us for 64 of 5 (128 channels); at 256 channels off 16 bytes,
// 8 loads to a row, they spill: 64 of one token 4.5 instead of 4.3 us, of 5 6.8 instead of 6.6 us.
template <typename T, int D, bool kWide>
struct PlainRow {
    static constexpr int W = D / 64;
    static constexpr int kAhead = D == 256 && !kWide ? 2 : 4;
    const u16* x;
    i64 stride;
    __device__ __forceinline__ PlainRow(const AppendArgs& a, u32 head, u32 side, u32 token)
        : x(static_cast<const u16*>(a.x[side]) + static_cast<i64>(token) * a.stride_token[side] +
            static_cast<i64>(head) * a.stride_head[side] + (threadIdx.x & 31u) * 2 * W),
          stride(a.stride_token[side])
    {
    }
    __device__ __forceinline__ void operator()(u32 t, float2 (&y)[W]) const
    {
        u32 raw[W];
        load_row<W, kWide>(x + t * stride, raw);
#pragma unroll
        for (int w = 0; w < W; ++w) y[w] = Pair<T>::floats(raw[w]);
    }
};

// The new tokens of a block, head and side as they are.
template <typename T, int D, bool kWide>
__device__ __forceinline__ void append_plain(const AppendArgs& a, u32 head, u32 side, u32 token, int page, u32 slot,
                                             u32 count)
{
    if (count < a.c.block || !append_full<T, D, kWide>(a, head, side, token, page))
        append_block<D>(a, head, side, page, slot, count, PlainRow<T, D, kWide>(a, head, side, token));
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

// A lane's token of a chunk of up to 32: whether it is the first new one of a block that is there,
// and the block.
struct Lead {
    bool leads;
    int page;
    u32 slot, count;  // tokens that the block held before, new ones
};

__device__ __forceinline__ Lead lead_of(const AppendArgs& a, u32 chunk)
{
    const u32 lane = threadIdx.x & 31u;
    const i64 token = static_cast<i64>(chunk) * a.chunk + lane;
    bool leads = lane < a.chunk && token < a.tokens;
    int page = -1;
    u32 slot = 0, count = 0, seq_first = 0, seq_last = 0;
    if (a.offsets) {  // sequences of the chunk's first and last token
        const i64 base = static_cast<i64>(chunk) * a.chunk;
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
    return Lead{leads, page, slot, count};
}

}  // namespace
}  // namespace hbfb
