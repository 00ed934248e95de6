// kv_rotary.cu -- new tokens into the 8-bit paged cache with keys and queries
// turned by their positions (kv_v1.h).
//
// A CTA takes a chunk of tokens.  It makes the cosines and sines of all pairs
// once, in shared memory, and its warps turn rows with them: eight heads of a
// token's queries at a time, and the blocks that begin in the chunk, a warp per
// head and side as in kv_append.cu.  The keys never exist in 16 bits: a block of
// new tokens alone is read and turned twice, for the largest magnitude and for the
// stored values (the second time from the L1 cache).  Products and
// sums are rounded one by one, so that what is stored does not depend on how a
// compiler joins them.
#include "kv_append.cuh"

namespace hbfb {
namespace {

constexpr u32 kRotaryWarps = 4;
constexpr u32 kRotaryHeads = 8;  // query heads of a token that a warp has in registers
constexpr u32 kMaxAxes = 4;

struct RotaryArgs {
    AppendArgs a;  // `wide`: k, v and q
    const void* q;
    i64 q_token, q_head;
    void* q_out;
    const int* positions;
    i64 positions_stride;
    const double* freq;
    const u8* axis;
    u32 q_heads, axes, pairs;
    bool append;  // whether any block is there
};

// sin and cos in 64 bits, rounded to 32.  Cody and Waite's reduction by multiples of pi/2 in two
// parts (exact up to 2^30 with fused products), then Taylor's series on [-pi/4, pi/4]: terms up to
// x^15, whose remainder is below 2e-15.
__device__ __forceinline__ void sine(double angle, float& sin32, float& cos32)
{
    double s, c;
    if (fabs(angle) < 1073741824.0) {
        const double k = rint(angle * 0.63661977236758134);  // 2 / pi
        double r = fma(-k, 1.5707963267948966, angle);       // pi / 2 ...
        r = fma(-k, 6.123233995736766e-17, r);               // ... and the rest of it
        const double z = r * r;
        s = fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 1307674368000.0, 1.0 / 6227020800.0), -1.0 / 39916800.0),
                                     1.0 / 362880.0), -1.0 / 5040.0), 1.0 / 120.0), -1.0 / 6.0);
        s = fma(r * z, s, r);
        c = fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 87178291200.0, 1.0 / 479001600.0), -1.0 / 3628800.0),
                                     1.0 / 40320.0), -1.0 / 720.0), 1.0 / 24.0), -0.5);
        c = fma(z, c, 1.0);
        const int quarter = static_cast<int>(k);
        const double t = s;
        if (quarter & 1) {
            s = c;
            c = t;
        }
        if (quarter & 2) s = -s;
        if ((quarter + 1) & 2) c = -c;
    } else {
        sincos(angle, &s, &c);  // frequencies above 1 at far positions, or not finite
    }
    sin32 = static_cast<float>(s);
    cos32 = static_cast<float>(c);
}

// What a lane needs to turn its channels of a row: its cosines and (signed) sines for a token.
template <int D, bool kNeighbours>
struct Turn {
    static constexpr int W = D / 64;
    bool turns;   // whether the lane's channels are among the pairs
    u32 first;    // its first pair
    int partner;  // the lane that has the other channels
    bool minus;
    float c[2 * W], s[2 * W];

    __device__ __forceinline__ explicit Turn(u32 pairs)
    {
        const u32 lane = threadIdx.x & 31u;
        if constexpr (kNeighbours) {
            turns = lane < pairs / W;
            first = turns ? lane * W : 0;
            partner = static_cast<int>(lane);
            minus = false;
        } else {
            const u32 lanes = pairs / (2 * W);
            turns = lane < 2 * lanes;
            minus = lane < lanes;
            partner = static_cast<int>(!turns ? lane : minus ? lane + lanes : lane - lanes);
            first = turns ? (minus ? lane : lane - lanes) * 2 * W : 0;
        }
    }

    __device__ __forceinline__ void load(const float* cosines, const float* sines)
    {
        constexpr int N = kNeighbours ? W : 2 * W;
        float x[N], y[N];
        read<N>(cosines + first, x);
        read<N>(sines + first, y);
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
            c[i] = x[kNeighbours ? i / 2 : i];
            s[i] = y[kNeighbours ? i / 2 : i];
            if (kNeighbours ? i % 2 == 0 : minus) s[i] = -s[i];
        }
    }

    // A row's channels of the lane, turned, in 32 bits.
    template <typename T>
    __device__ __forceinline__ void apply(const u32 (&raw)[W], float2 (&y)[W]) const
    {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 x = Pair<T>::floats(raw[w]);
            float2 p = make_float2(x.y, x.x);
            if constexpr (!kNeighbours) p = Pair<T>::floats(__shfl_sync(0xffffffffu, raw[w], partner));
            y[w].x = __fadd_rn(__fmul_rn(x.x, c[2 * w]), __fmul_rn(p.x, s[2 * w]));
            y[w].y = __fadd_rn(__fmul_rn(x.y, c[2 * w + 1]), __fmul_rn(p.y, s[2 * w + 1]));
            if (!turns) y[w] = x;
        }
    }

private:
    template <int N>
    static __device__ __forceinline__ void read(const float* from, float (&x)[N])
    {
        if constexpr (N == 1) {
            x[0] = *from;
        } else if constexpr (N == 2) {
            const float2 y = *reinterpret_cast<const float2*>(from);
            x[0] = y.x;
            x[1] = y.y;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 y = *reinterpret_cast<const float4*>(from + i);
                x[i] = y.x;
                x[i + 1] = y.y;
                x[i + 2] = y.z;
                x[i + 3] = y.w;
            }
        }
    }
};

__device__ __forceinline__ u32 packed(float2 x, __nv_bfloat16)
{
    const __nv_bfloat162 y = __float22bfloat162_rn(x);
    return *reinterpret_cast<const u32*>(&y);
}
__device__ __forceinline__ u32 packed(float2 x, __half)
{
    const __half2 y = __float22half2_rn(x);
    return *reinterpret_cast<const u32*>(&y);
}

template <int W>
__device__ __forceinline__ void store_row(u16* to, const u32 (&x)[W])
{
    if constexpr (W == 1) *reinterpret_cast<u32*>(to) = x[0];
    else if constexpr (W == 2) *reinterpret_cast<uint2*>(to) = make_uint2(x[0], x[1]);
    else *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
}

// The cosines and sines in shared memory: [tokens of the CTA][pairs] each.
struct Circle {
    const float* cosines;
    const float* sines;
    u32 pairs;
};

// A head's new keys, turned: the `row` of append_block; `circle` begins with the block's first new
// token.
template <typename T, int D, bool kWide, bool kNeighbours>
struct TurnedRow {
    static constexpr int W = D / 64;
    const u16* x;
    i64 stride;
    Circle circle;
    __device__ __forceinline__ void operator()(u32 t, float2 (&y)[W]) const
    {
        u32 raw[W];
        load_row<W, kWide>(x + t * stride, raw);
        Turn<D, kNeighbours> turn(circle.pairs);
        turn.load(circle.cosines + t * circle.pairs, circle.sines + t * circle.pairs);
        turn.template apply<T>(raw, y);
    }
};

// A head's keys of a block whose tokens are all new, by one warp; false, with nothing written, where
// a turned element is not finite.  Rounding keeps the order, so the least and greatest of a channel
// give its bounds.
template <typename T, int D, bool kWide, bool kNeighbours>
__device__ __forceinline__ bool append_full_turned(const AppendArgs& a, u32 head, u32 token, int page,
                                                   const Circle& circle)
{
    constexpr int W = D / 64;
    const u32 lane = threadIdx.x & 31u, block = a.c.block;
    const i64 stride = a.stride_token[0];
    const u16* x = static_cast<const u16*>(a.x[0]) + static_cast<i64>(token) * stride +
                   static_cast<i64>(head) * a.stride_head[0] + lane * 2 * W;
    const u64 at = (static_cast<u64>(page) * a.c.heads + head) * 2;
    constexpr u32 R = 8;  // rows at a time
    u32 raw[R][W];
    float2 lo[W], hi[W];
    auto load_rows = [&](u32 row0) {
#pragma unroll
        for (u32 r = 0; r < R; ++r) load_row<W, kWide>(x + (row0 + r) * stride, raw[r]);
    };
    Turn<D, kNeighbours> turn(circle.pairs);
    auto turned = [&](u32 row0, u32 r, float2 (&y)[W]) {
        turn.load(circle.cosines + (row0 + r) * circle.pairs, circle.sines + (row0 + r) * circle.pairs);
        turn.template apply<T>(raw[r], y);
    };
    load_rows(0);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        lo[w] = make_float2(3.402823466e38f, 3.402823466e38f);
        hi[w] = make_float2(-3.402823466e38f, -3.402823466e38f);
    }
    bool finite = true;
    for (u32 row0 = 0;;) {
#pragma unroll
        for (u32 r = 0; r < R; ++r) {
            float2 y[W];
            turned(row0, r, y);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                finite &= fabsf(y[w].x) <= 3.402823466e38f && fabsf(y[w].y) <= 3.402823466e38f;
                lo[w] = make_float2(fminf(lo[w].x, y[w].x), fminf(lo[w].y, y[w].y));
                hi[w] = make_float2(fmaxf(hi[w].x, y[w].x), fmaxf(hi[w].y, y[w].y));
            }
        }
        row0 += R;
        if (row0 == block) break;
        load_rows(row0);
    }
    if (!__all_sync(0xffffffffu, finite)) return false;
    float most = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
        most = fmaxf(most, fmaxf(fmaxf(fabsf(lo[w].x), fabsf(lo[w].y)), fmaxf(fabsf(hi[w].x), fabsf(hi[w].y))));
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float now = kv_power(scale_exponent(most)), inverse = 1.0f / now;
    if (lane == 0) a.c.scale[at] = now;
    auto stored = [&](float2 y) { return store_e4m3(make_float2(y.x * inverse, y.y * inverse)); };
    u8* out = a.c.data + at * block * D + lane * 2 * W;
    for (u32 row0 = 0;;) {
        load_rows(row0);
#pragma unroll
        for (u32 r = 0; r < R; ++r) {
            float2 y[W];
            u32 b[W];
            turned(row0, r, y);
#pragma unroll
            for (int w = 0; w < W; ++w) b[w] = stored(y[w]);
            put_row<W>(out + (row0 + r) * D, b);
        }
        row0 += R;
        if (row0 == block) break;
    }
    u32 least[W], greatest[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        least[w] = stored(lo[w]);
        greatest[w] = stored(hi[w]);
    }
    put_bounds<D>(a, page, head, least, greatest);
    return true;
}

// Heads [head0, head0 + kRotaryHeads) of a token's queries by one warp.
template <typename T, int D, bool kWide, bool kNeighbours>
__device__ __forceinline__ void turn_queries(const RotaryArgs& r, u32 token, u32 head0, const Circle& circle)
{
    constexpr int W = D / 64;
    const u32 lane = threadIdx.x & 31u;
    const u16* x = static_cast<const u16*>(r.q) + static_cast<i64>(token) * r.q_token + lane * 2 * W;
    u16* out = static_cast<u16*>(r.q_out) + (static_cast<u64>(token) * r.q_heads + head0) * D + lane * 2 * W;
    u32 raw[kRotaryHeads][W];
#pragma unroll
    for (u32 h = 0; h < kRotaryHeads; ++h) {
        if (head0 + h < r.q_heads) {
            load_row<W, kWide>(x + static_cast<i64>(head0 + h) * r.q_head, raw[h]);
        } else {
#pragma unroll
            for (int w = 0; w < W; ++w) raw[h][w] = 0;
        }
    }
    Turn<D, kNeighbours> turn(circle.pairs);
    turn.load(circle.cosines, circle.sines);
#pragma unroll
    for (u32 h = 0; h < kRotaryHeads; ++h) {
        float2 y[W];
        u32 b[W];
        turn.template apply<T>(raw[h], y);
#pragma unroll
        for (int w = 0; w < W; ++w) b[w] = packed(y[w], T{});
        if (head0 + h < r.q_heads) store_row<W>(out + h * D, b);
    }
}

template <typename T, int D, bool kWide, bool kNeighbours>
__global__ void __launch_bounds__(kRotaryWarps * 32, D == 256 ? 3 : 6) rotary_kernel(const RotaryArgs r)
{
    extern __shared__ float4 shared[];
    const AppendArgs& a = r.a;
    const u32 base = blockIdx.x * a.chunk, mine = min(a.chunk, a.tokens - base), pairs = r.pairs;
    const Lead lead = r.append ? lead_of(a) : Lead{false, -1, 0, 0};
    const u32 leads = __ballot_sync(0xffffffffu, lead.leads);
    // tokens of the chunk, and those behind it of blocks that begin in it
    const u32 all = max(mine, __reduce_max_sync(0xffffffffu, lead.leads ? (threadIdx.x & 31u) + lead.count : 0));
    float* cosines = reinterpret_cast<float*>(shared);
    float* sines = cosines + all * pairs;
    for (u32 i = threadIdx.x; i < all * pairs; i += blockDim.x) {
        const u32 token = i / pairs, pair = i - token * pairs;
        const u32 axis = min(static_cast<u32>(r.axis[pair]), r.axes - 1);
        const int position = r.positions[static_cast<i64>(axis) * r.positions_stride + base + token];
        sine(__dmul_rn(static_cast<double>(position), r.freq[pair]), sines[i], cosines[i]);
    }
    __syncthreads();
    // warps share the blocks' heads and sides, then the tokens' heads
    const u32 sides = a.c.heads * 2, blocks = __popc(leads) * sides;
    const u32 groups = (r.q_heads + kRotaryHeads - 1) / kRotaryHeads, total = blocks + mine * groups;
    for (u32 u = blockIdx.y * kRotaryWarps + (threadIdx.x >> 5); u < total; u += gridDim.y * kRotaryWarps) {
        if (u >= blocks) {
            const u32 token = (u - blocks) / groups, head0 = ((u - blocks) - token * groups) * kRotaryHeads;
            turn_queries<T, D, kWide, kNeighbours>(r, base + token, head0,
                                                   Circle{cosines + token * pairs, sines + token * pairs, pairs});
            continue;
        }
        const u32 which = u / sides, head = (u - which * sides) >> 1, side = u & 1u;  // `sides` is even
        u32 left = leads;
        for (u32 i = 0; i < which; ++i) left &= left - 1;
        const int who = __ffs(left) - 1;
        const int page = __shfl_sync(0xffffffffu, lead.page, who);
        const u32 slot = __shfl_sync(0xffffffffu, lead.slot, who), count = __shfl_sync(0xffffffffu, lead.count, who);
        const u32 token = base + static_cast<u32>(who);
        if (side) {
            append_plain<T, D, kWide>(a, head, side, token, page, slot, count);
            continue;
        }
        const Circle circle{cosines + static_cast<u32>(who) * pairs, sines + static_cast<u32>(who) * pairs, pairs};
        if (count < a.c.block || !append_full_turned<T, D, kWide, kNeighbours>(a, head, token, page, circle)) {
            const PlainRow<T, D, kWide> from(a, head, 0, token);
            append_block<D>(a, head, 0, page, slot, count,
                            TurnedRow<T, D, kWide, kNeighbours>{from.x, from.stride, circle});
        }
    }
}

template <typename T, int D, bool kWide, bool kNeighbours>
bool launch(const RotaryArgs& r, u32 spread, cudaStream_t s)
{
    const u32 smem = (r.a.chunk - 1 + r.a.c.block) * r.pairs * 8;
    constexpr u32 kMost = (15 + 64) * (D / 2) * 8;
    static std::atomic<u64> seen{0};
    if (smem > 48 * 1024 && !kv_allow_smem(rotary_kernel<T, D, kWide, kNeighbours>, kMost, seen)) return false;
    const dim3 grid((r.a.tokens + r.a.chunk - 1) / r.a.chunk, spread);
    return kv_launch(rotary_kernel<T, D, kWide, kNeighbours>, grid, kRotaryWarps * 32, s, smem, 1, false, r);
}

template <typename T, int D>
bool launch_wide(const RotaryArgs& r, u32 spread, bool neighbours, cudaStream_t s)
{
    if (r.a.wide) return neighbours ? launch<T, D, true, true>(r, spread, s) : launch<T, D, true, false>(r, spread, s);
    return neighbours ? launch<T, D, false, true>(r, spread, s) : launch<T, D, false, false>(r, spread, s);
}

template <typename T>
bool launch_dim(const RotaryArgs& r, u32 spread, bool neighbours, cudaStream_t s)
{
    switch (r.a.c.dim) {
    case 64: return launch_wide<T, 64>(r, spread, neighbours, s);
    case 128: return launch_wide<T, 128>(r, spread, neighbours, s);
    default: return launch_wide<T, 256>(r, spread, neighbours, s);
    }
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" int hbfsim_kv_append_rotary_v1(const hbfsim_kv_cache_v1* cache, const hbfsim_kv_append_batch_v1* b,
                                          const hbfsim_kv_rotary_v1* x, void* stream)
{
    RotaryArgs r{};
    AppendArgs& a = r.a;
    if (const int rc = append_check(cache, b, a)) return rc;
    if (!x || x->struct_size != sizeof(*x) || x->version != HBFSIM_KV_V1_VERSION || x->neighbours > 1 ||
        x->q_heads > (1u << 16) || x->axes == 0 || x->axes > kMaxAxes)
        return HBFSIM_INVALID_ARGUMENT;
    // pairs: whole lanes of channels, so that a channel's partner is a whole lane away
    if (x->pairs == 0 || x->pairs > cache->head_dim / 2 || x->pairs % (cache->head_dim / 32))
        return HBFSIM_UNSUPPORTED;
    if (b->tokens == 0) return HBFSIM_OK;
    if (!x->positions || !x->freq || !x->axis || (x->q_heads && (!x->q || !x->q_out)))
        return HBFSIM_INVALID_ARGUMENT;
    if (!kv_aligned(x->q, 2) || !kv_aligned(x->q_out, 16) || !kv_aligned(x->positions, 4) || !kv_aligned(x->freq, 8))
        return HBFSIM_INVALID_ARGUMENT;
    r.append = b->width != 0 && a.c.pages != 0;
    if (!r.append && x->q_heads == 0) return HBFSIM_OK;
    r.q = x->q;
    r.q_token = x->q_stride_token;
    r.q_head = x->q_stride_head;
    r.q_out = x->q_out;
    r.positions = x->positions;
    r.positions_stride = x->positions_stride;
    r.freq = x->freq;
    r.axis = x->axis;
    r.q_heads = x->q_heads;
    r.axes = x->axes;
    r.pairs = x->pairs;
    a.wide = a.wide && (x->q_heads == 0 || kv_rows_wide(x->q, x->q_stride_token, x->q_stride_head));
    // warps' work of a token: groups of query heads, and its share of the blocks' heads and sides
    const u32 groups = (r.q_heads + kRotaryHeads - 1) / kRotaryHeads, sides = a.c.heads * 2;
    a.chunk = 1;
    while (a.chunk < 16 &&
           static_cast<u64>(a.tokens) * (groups + sides) > static_cast<u64>(a.chunk) * 16 * kv_sm_count())
        a.chunk *= 2;
    const u32 spread = std::max(1u, (groups + sides + kRotaryWarps * a.chunk - 1) / (kRotaryWarps * a.chunk));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool ok = b->type == HBFSIM_KV_BF16 ? launch_dim<__nv_bfloat16>(r, spread, x->neighbours != 0, s)
                                              : launch_dim<__half>(r, spread, x->neighbours != 0, s);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
