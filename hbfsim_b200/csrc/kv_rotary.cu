// kv_rotary.cu -- new tokens into the 8-bit paged cache with keys and queries
// turned by their positions (kv_v1.h).
//
// One launch, three kinds of CTA.  Keys: a chunk of tokens as in kv_append.cu, whose
// blocks' cosines and sines are made once, in shared memory; a warp turns up to 16 of
// a head's rows of a block twice, for the largest magnitude and for the stored values
// (the second time from the caches), so the keys never exist in 16 bits; blocks of 32
// or 64 tokens are shared by two or four warps (2,000 tokens in blocks of 64 took 99
// us by one, 30 us by four).  Values: as in kv_append.cu.  Queries: every warp by
// itself.  It takes a token's heads, asks for the first rows, makes the token's
// cosines and sines meanwhile, and reads the next rows while it turns the ones at
// hand.  Keys and values come first: their CTAs take longest (mixed with the queries'
// the call took as long).  Products and sums are rounded one by one, so that what is
// stored does not depend on how a compiler joins them.
//
// Prompts of 31,668 tokens in all (32 query and 8 key/value heads of 128 channels)
// take 134 us, 718 MB of input, queries and blocks at 5.4 TB/s, 82 % of a copy's rate:
// the queries alone 80 us (6.5 TB/s, a copy's rate), the keys and values alone 74 us,
// where warps wait for their rows at 53 % of the issue slots.  Rows off 16 bytes, of q,
// k or v, take 181 us by loads of 2 bytes.  A step's 64 tokens take 5.8 us: a launch,
// the chain of reads of an append, the positions and one turn of 64-bit arithmetic.
#include "kv_append.cuh"

namespace hbfb {
namespace {

constexpr u32 kRotaryWarps = 4;
constexpr u32 kRotaryHeads = 8;  // query heads that a warp reads at a time
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
    // thread blocks for keys, then for values, so many to a chunk; the others are for queries
    u32 key_blocks, key_spread, value_blocks, value_spread;
    u32 parts, part;  // warps to a token's queries, groups of heads of each
};

// sin and cos in 64 bits, rounded to 32.  Cody and Waite's reduction by multiples of pi/2 in two
// parts (exact up to 2^30 with fused products), then Taylor's series on [-pi/4, pi/4]: terms up to
// x^15, whose remainder is below 2e-15.
__device__ __forceinline__ void sine(double angle, float& sin32, float& cos32)
{
    double s, c;
    if (fabs(angle) < 1073741824.0) {
        // the nearest whole number of quarter turns: added to 1.5 * 2^52, it is the sum's last bits
        const double shifted = fma(angle, 0.63661977236758134, 6755399441055744.0);  // 2 / pi
        const double k = shifted - 6755399441055744.0;
        const int quarter = __double2loint(shifted);
        double r = fma(-k, 1.5707963267948966, angle);  // pi / 2 ...
        r = fma(-k, 6.123233995736766e-17, r);          // ... and the rest of it
        const double z = r * r;
        s = fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 1307674368000.0, 1.0 / 6227020800.0), -1.0 / 39916800.0),
                                     1.0 / 362880.0), -1.0 / 5040.0), 1.0 / 120.0), -1.0 / 6.0);
        s = fma(r * z, s, r);
        c = fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 87178291200.0, 1.0 / 479001600.0), -1.0 / 3628800.0),
                                     1.0 / 40320.0), -1.0 / 720.0), 1.0 / 24.0), -0.5);
        c = fma(z, c, 1.0);
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

__device__ __forceinline__ void circle_at(const RotaryArgs& r, u32 token, u32 pair, float& sin32, float& cos32)
{
    const u32 axis = min(static_cast<u32>(r.axis[pair]), r.axes - 1);
    const int position = r.positions[static_cast<i64>(axis) * r.positions_stride + token];
    sine(__dmul_rn(static_cast<double>(position), r.freq[pair]), sin32, cos32);
}

// Two products in 32 bits at once; sums one by one: a sum of two at once after them is joined with
// a product into one rounding, whatever the instructions say.
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(r)
        : "l"(*reinterpret_cast<u64*>(&a)), "l"(*reinterpret_cast<u64*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b)
{
    return make_float2(__fsub_rn(a.x, b.x), __fsub_rn(a.y, b.y));
}

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

// N words of two elements, or N pairs of numbers.
template <int N>
__device__ __forceinline__ void store_words(u16* to, const u32 (&x)[N])
{
    if constexpr (N == 1) *reinterpret_cast<u32*>(to) = x[0];
    else if constexpr (N == 2) *reinterpret_cast<uint2*>(to) = make_uint2(x[0], x[1]);
    else *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
}
template <int N>
__device__ __forceinline__ void load_floats(const float* from, float2 (&x)[N])
{
    if constexpr (N == 1) {
        x[0] = *reinterpret_cast<const float2*>(from);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float4 y = *reinterpret_cast<const float4*>(from + 2 * i);
            x[i] = make_float2(y.x, y.y);
            x[i + 1] = make_float2(y.z, y.w);
        }
    }
}

// Half a warp takes a row: a lane has V neighbouring pairs, that is, V channels at `lo` and V at
// `hi`.  Channels i and i + pairs are in one lane that way, and a warp turns two rows at once.
// Lanes past the pairs carry the channels that stay.
enum Layout { kSplit, kNeighbours, kWhole };  // i with i + pairs; 2i with 2i + 1; i with i + D / 2
template <int D, int kLayout>
struct Lane {
    static constexpr int V = D / 32, N = V / 2;
    u32 lo, hi, pair;
    bool turns;

    __device__ __forceinline__ explicit Lane(u32 pairs)
    {
        pair = (threadIdx.x & 15u) * V;
        turns = kLayout == kWhole || pair < pairs;
        lo = kLayout == kNeighbours || !turns ? 2 * pair : pair;
        hi = lo + (kLayout == kWhole ? D / 2 : kLayout == kNeighbours || !turns ? V : pairs);
        if (!turns) pair = 0;
    }

    struct Circle {
        float2 c[N], s[N];
    };
    __device__ __forceinline__ void load(const float* cosines, const float* sines, Circle& a) const
    {
        load_floats<N>(cosines + pair, a.c);
        load_floats<N>(sines + pair, a.s);
    }
    // The same made here: the two lanes that turn by the same pairs make half of them each.
    __device__ __forceinline__ void make(const RotaryArgs& r, u32 token, Circle& a) const
    {
        const u32 half = (threadIdx.x & 31u) >> 4;
        float c[N], s[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            c[i] = s[i] = 0.0f;
            if (turns) circle_at(r, token, pair + half * N + i, s[i], c[i]);
        }
        float* all_c = reinterpret_cast<float*>(a.c);
        float* all_s = reinterpret_cast<float*>(a.s);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float oc = __shfl_xor_sync(0xffffffffu, c[i], 16), os = __shfl_xor_sync(0xffffffffu, s[i], 16);
            all_c[i] = half ? oc : c[i];
            all_c[N + i] = half ? c[i] : oc;
            all_s[i] = half ? os : s[i];
            all_s[N + i] = half ? s[i] : os;
        }
    }

    // The lane's channels at lo (x) and hi (y) in 32 bits, turned.
    template <typename T>
    __device__ __forceinline__ void apply(const u32 (&low)[N], const u32 (&high)[N], const Circle& a, float2 (&x)[N],
                                          float2 (&y)[N]) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = Pair<T>::floats(low[i]);
            y[i] = Pair<T>::floats(high[i]);
        }
        if (!turns) return;
        if constexpr (kLayout == kNeighbours) {
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) {  // pairs of channels, N at lo and N at hi
                const float c = i & 1 ? a.c[i / 2].y : a.c[i / 2].x, s = i & 1 ? a.s[i / 2].y : a.s[i / 2].x;
                float2& p = i < N ? x[i % N] : y[i % N];
                p = make_float2(__fsub_rn(__fmul_rn(p.x, c), __fmul_rn(p.y, s)),
                                __fadd_rn(__fmul_rn(p.x, s), __fmul_rn(p.y, c)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 m = sub2(mul2(x[i], a.c[i]), mul2(y[i], a.s[i]));
                y[i] = add2(mul2(x[i], a.s[i]), mul2(y[i], a.c[i]));
                x[i] = m;
            }
        }
    }
};

// The cosines and sines in shared memory: [tokens of the CTA][pairs] each.
struct Table {
    const float* cosines;
    const float* sines;
    u32 pairs;
};

// A head's new keys, turned: the `row` of append_block, a lane's channels side by side; `table`
// begins with the block's first new token.
template <typename T, int D, bool kWide, int kLayout>
struct TurnedRow {
    static constexpr int W = D / 64;
    static constexpr int kAhead = 4;
    const u16* x;  // the lane's channels of the first token
    i64 stride;
    Table table;
    __device__ __forceinline__ void operator()(u32 t, float2 (&y)[W]) const
    {
        const u32 channel = (threadIdx.x & 31u) * 2 * W, pairs = table.pairs;
        const bool turns = channel < 2 * pairs, second = channel >= pairs;
        const u32 pair = !turns ? 0 : kLayout == kNeighbours ? channel / 2 : second ? channel - pairs : channel;
        const float* c = table.cosines + t * pairs + pair;
        const float* s = table.sines + t * pairs + pair;
        u32 raw[W], other[W];
        load_row<W, kWide>(x + t * stride, raw);
        const int apart = static_cast<int>(pairs);
        const int away = kLayout == kNeighbours || !turns ? 0 : second ? -apart : apart;
        load_row<W, kWide>(x + t * stride + away, other);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            y[w] = Pair<T>::floats(raw[w]);
            if (!turns) continue;
            float2 p = Pair<T>::floats(other[w]), cc, ss;
            if constexpr (kLayout == kNeighbours) {
                p = make_float2(p.y, p.x);
                cc = make_float2(c[w], c[w]);
                ss = make_float2(-s[w], s[w]);
            } else {
                cc = make_float2(c[2 * w], c[2 * w + 1]);
                ss = make_float2(s[2 * w], s[2 * w + 1]);
                if (!second) ss = make_float2(-ss.x, -ss.y);
            }
            y[w] = add2(mul2(y[w], cc), mul2(p, ss));
        }
    }
};

// The lesser and the greater of two, NaN if either is.
__device__ __forceinline__ float least_of(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float greatest_of(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// N words of two stored values, as put_row writes them.
template <int N>
__device__ __forceinline__ void load_values(const u8* from, u32 (&b)[N])
{
    if constexpr (N == 1) {
        b[0] = *reinterpret_cast<const u16*>(from);
    } else if constexpr (N == 2) {
        const u32 x = *reinterpret_cast<const u32*>(from);
        b[0] = x & 0xffffu;
        b[1] = x >> 16;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(from);
        b[0] = x.x & 0xffffu;
        b[1] = x.x >> 16;
        b[2] = x.y & 0xffffu;
        b[3] = x.y >> 16;
    }
}

// A head's keys of a block by one warp, a row at a time.
template <typename T, int D, bool kWide, int kLayout>
__device__ __forceinline__ void append_rows(const AppendArgs& a, u32 head, u32 token, int page, u32 slot, u32 count,
                                            const Table& table)
{
    const PlainRow<T, D, kWide> from(a, head, 0, token);
    append_block<D>(a, head, 0, page, slot, count, TurnedRow<T, D, kWide, kLayout>{from.x, from.stride, table});
}

// Where the warps that share a block meet: each 16 of its rows.
template <int D>
struct Join {
    float most[kRotaryWarps];
    float ends[kRotaryWarps][2][D];  // least and greatest of the channels
};

// A head's keys of a block by `parts` warps (block / 16 of them), of which this is the part-th; all
// warps of the CTA come here, the same number of times.  Rounding keeps the order, so the least and
// greatest of a channel give its bounds.  `table` begins with the block's first new token.  False, with
// nothing written, where a turned element is not finite.
template <typename T, int D, bool kWide, int kLayout>
__device__ __forceinline__ bool append_turned(const AppendArgs& a, bool active, u32 head, u32 token, int page, u32 slot,
                                              u32 count, u32 part, u32 parts, const Table& table, Join<D>& join)
{
    using Of = Lane<D, kLayout>;
    constexpr int N = Of::N;
    constexpr u32 R = 2;  // steps of two rows at a time
    const Of mine(table.pairs);
    const u32 lane = threadIdx.x & 31u, half = lane >> 4, warp = threadIdx.x >> 5, block = a.c.block;
    const u64 at = (static_cast<u64>(page) * a.c.heads + head) * 2;
    u8* out = a.c.data + at * block * D;
    // the warp's rows: [first, held) are there already, [from, to) are new
    const u32 first = part * 16, from = max(slot, first), to = active ? min(slot + count, first + 16) : 0;
    const u32 held = min(slot, first + 16);
    const bool full = from + 16 == to;  // of new ones: the rows' places are plain then
    const i64 stride = a.stride_token[0];
    const u16* x = static_cast<const u16*>(a.x[0]) + (static_cast<i64>(token) - slot) * stride +
                   static_cast<i64>(head) * a.stride_head[0];
    // Turned: the channels at mine.lo and at mine.hi.  16 rows kept from the first time on, with 16
    // warps on an SM, took 149 us for prompts that take 143 with 8 rows at a time (20 warps) and 139
    // with 4 (24 warps), in chunks of 16 tokens.
    float2 y[R][2][N];
    auto turn_rows = [&](u32 row0, auto plain_rows) {
        constexpr bool kPlain = decltype(plain_rows)::value;
        auto row_at = [&](u32 r) {  // past the end: the last again
            return kPlain ? row0 + 2 * r + half : min(row0 + 2 * r + half, to - 1);
        };
        u32 low[R][N], high[R][N];
#pragma unroll
        for (u32 r = 0; r < R; ++r) {
            load_row<N, kWide>(x + row_at(r) * stride + mine.lo, low[r]);
            load_row<N, kWide>(x + row_at(r) * stride + mine.hi, high[r]);
        }
#pragma unroll
        for (u32 r = 0; r < R; ++r) {
            typename Of::Circle circle;
            const u32 row = (row_at(r) - slot) * table.pairs;
            mine.load(table.cosines + row, table.sines + row, circle);
            mine.template apply<T>(low[r], high[r], circle, y[r][0], y[r][1]);
        }
    };
    const float was = active && slot ? a.c.scale[at] : 0.0f;  // written only after all have met
    constexpr float kMost = 3.402823466e38f;
    float2 lo[2][N], hi[2][N];  // least and greatest of the channels
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            lo[k][i] = make_float2(kMost, kMost);
            hi[k][i] = make_float2(-kMost, -kMost);
        }
    auto span = [&](int k, int i, float2 z) {
        lo[k][i] = make_float2(least_of(lo[k][i].x, z.x), least_of(lo[k][i].y, z.y));
        hi[k][i] = make_float2(greatest_of(hi[k][i].x, z.x), greatest_of(hi[k][i].y, z.y));
    };
    auto find_ends = [&](auto plain_rows) {
#pragma unroll 1
        for (u32 row0 = from; row0 < to; row0 += 2 * R) {
            turn_rows(row0, plain_rows);
#pragma unroll
            for (u32 r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) span(k, i, y[r][k][i]);
        }
    };
    if (full) find_ends(std::true_type{});
    else find_ends(std::false_type{});
    float most = 0.0f;  // NaN if any is
    if (from < to) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i)
                most = greatest_of(most, greatest_of(greatest_of(fabsf(lo[k][i].x), fabsf(lo[k][i].y)),
                                                     greatest_of(fabsf(hi[k][i].x), fabsf(hi[k][i].y))));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = greatest_of(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (parts > 1) {
        if (lane == 0) join.most[warp] = most;
        __syncthreads();
        for (u32 i = 0; i < parts; ++i) most = greatest_of(most, join.most[warp - part + i]);
    }
    const bool plain = most <= kMost;
    const float now = fmaxf(kv_power(scale_exponent(plain ? most : 0.0f)), was), inverse = 1.0f / now;
    auto store_rows = [&](auto plain_rows) {
        constexpr bool kPlain = decltype(plain_rows)::value;
#pragma unroll 1
        for (u32 row0 = from; row0 < to; row0 += 2 * R) {
            turn_rows(row0, plain_rows);
#pragma unroll
            for (u32 r = 0; r < R; ++r) {
                u32 b[2][N];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) b[k][i] = store_e4m3(mul2(y[r][k][i], make_float2(inverse, inverse)));
                const u32 row = row0 + 2 * r + half;
                if (kPlain || row < to) {
                    put_row<N>(out + row * D + mine.lo, b[0]);
                    put_row<N>(out + row * D + mine.hi, b[1]);
                }
            }
        }
    };
    if (active && plain) {
        if (lane == 0 && part == 0) a.c.scale[at] = now;
        if (full) store_rows(std::true_type{});
        else store_rows(std::false_type{});
        const u32 none[N] = {};
        for (u32 row = max(slot + count, first) + half; row < first + 16; row += 2) {
            put_row<N>(out + row * D + mine.lo, none);
            put_row<N>(out + row * D + mine.hi, none);
        }
    }
    // from here on in units of the scale
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            lo[k][i] = mul2(lo[k][i], make_float2(inverse, inverse));
            hi[k][i] = mul2(hi[k][i], make_float2(inverse, inverse));
        }
    if (active && plain) {  // what the block held before: rounded again if the scale grew
        const float shrink = slot ? was / now : 1.0f;
        for (u32 row0 = first; row0 < held; row0 += 2 * R) {
            u32 b[R][2][N];
#pragma unroll
            for (u32 r = 0; r < R; ++r) {
                const u32 row = min(row0 + 2 * r + half, held - 1);
                load_values<N>(out + row * D + mine.lo, b[r][0]);
                load_values<N>(out + row * D + mine.hi, b[r][1]);
            }
            __syncwarp();  // the last row may be read by both halves
#pragma unroll
            for (u32 r = 0; r < R; ++r) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        float2 z = __half22float2(stored_f16(b[r][k][i]));
                        if (shrink != 1.0f) {
                            b[r][k][i] = store_e4m3(mul2(z, make_float2(shrink, shrink)));
                            z = __half22float2(stored_f16(b[r][k][i]));
                        }
                        span(k, i, make_float2(z.x == z.x ? z.x : 0.0f, z.y == z.y ? z.y : 0.0f));  // NaN counts as 0
                    }
                const u32 row = row0 + 2 * r + half;
                if (shrink != 1.0f && row < held) {
                    put_row<N>(out + row * D + mine.lo, b[r][0]);
                    put_row<N>(out + row * D + mine.hi, b[r][1]);
                }
            }
            __syncwarp();
        }
    }
    // the rows of both halves together: the lower half has the least, the upper one the greatest
    float2 ends[2][N];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 give = half ? lo[k][i] : hi[k][i], keep = half ? hi[k][i] : lo[k][i];
            float2 other;
            other.x = __shfl_xor_sync(0xffffffffu, give.x, 16);
            other.y = __shfl_xor_sync(0xffffffffu, give.y, 16);
            ends[k][i] = half ? make_float2(fmaxf(keep.x, other.x), fmaxf(keep.y, other.y))
                              : make_float2(fminf(keep.x, other.x), fminf(keep.y, other.y));
        }
    if (parts > 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i)
                *reinterpret_cast<float2*>(&join.ends[warp][half][(k ? mine.hi : mine.lo) + 2 * i]) = ends[k][i];
        __syncthreads();
        for (u32 w = warp + 1; part == 0 && w < warp + parts; ++w)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float* other = &join.ends[w][half][(k ? mine.hi : mine.lo) + 2 * i];
                    const float2 z = *reinterpret_cast<const float2*>(other), e = ends[k][i];
                    ends[k][i] = half ? make_float2(fmaxf(e.x, z.x), fmaxf(e.y, z.y))
                                      : make_float2(fminf(e.x, z.x), fminf(e.y, z.y));
                }
    }
    if (!active || part || !plain) return plain;
    std::int8_t* bound = a.c.bounds + (static_cast<u64>(page) * a.c.heads + head) * 2 * D + half * D;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 z = __half22float2(stored_f16(store_e4m3(ends[k][i])));
            const float2 q = make_float2(z.x * 0.25f, z.y * 0.25f);
            *reinterpret_cast<char2*>(bound + (k ? mine.hi : mine.lo) + 2 * i) =
                half ? make_char2(static_cast<signed char>(ceilf(q.x)), static_cast<signed char>(ceilf(q.y)))
                     : make_char2(static_cast<signed char>(floorf(q.x)), static_cast<signed char>(floorf(q.y)));
        }
    return true;
}

// `part` groups of heads of a token's queries by one warp.
template <typename T, int D, bool kWide, int kLayout>
__device__ __forceinline__ void turn_queries(const RotaryArgs& r, u32 token, u32 group)
{
    using Of = Lane<D, kLayout>;
    constexpr int N = Of::N;
    constexpr u32 R = kRotaryHeads / 2;
    const Of mine(r.pairs);
    const u32 half = (threadIdx.x & 31u) >> 4, end = min(r.q_heads, (group + r.part) * kRotaryHeads);
    u32 head = group * kRotaryHeads + half;  // the first of the lane's rows at hand
    const u16* x = static_cast<const u16*>(r.q) + static_cast<i64>(token) * r.q_token +
                   static_cast<i64>(head) * r.q_head + mine.lo;
    u16* out = static_cast<u16*>(r.q_out) + (static_cast<u64>(token) * r.q_heads + head) * D + mine.lo;
    const u32 away = mine.hi - mine.lo;
    const i64 two = 2 * r.q_head;
    u32 low[2][R][N], high[2][R][N];  // rows at hand, rows on their way
    auto load_rows = [&](u32 first, u32 (&l)[R][N], u32 (&h)[R][N]) {
#pragma unroll
        for (u32 i = 0; i < R; ++i) {
            if (first + 2 * i < end) {
                load_row<N, kWide>(x, l[i]);
                load_row<N, kWide>(x + away, h[i]);
            }
            x += two;
        }
    };
    load_rows(head, low[0], high[0]);
    typename Of::Circle circle;
    mine.make(r, token, circle);
    for (;;) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            load_rows(head + kRotaryHeads, low[1 - k], high[1 - k]);
#pragma unroll
            for (u32 i = 0; i < R; ++i) {
                float2 p[N], q[N];
                u32 b[2][N];
                mine.template apply<T>(low[k][i], high[k][i], circle, p, q);
#pragma unroll
                for (int w = 0; w < N; ++w) {
                    b[0][w] = packed(p[w], T{});
                    b[1][w] = packed(q[w], T{});
                }
                if (head + 2 * i < end) {
                    store_words<N>(out + 2 * i * D, b[0]);
                    store_words<N>(out + 2 * i * D + away, b[1]);
                }
            }
            head += kRotaryHeads;
            out += kRotaryHeads * D;
            if (head - half >= end) return;
        }
    }
}

// The block of a chunk's lead that a warp's `u`-th piece of work is in, `each` pieces to a block.
struct Piece {
    u32 who, head;
    int page;
    u32 slot, count;
};
__device__ __forceinline__ Piece piece_at(const Lead& lead, u32 leads, u32 u, u32 each)
{
    const u32 which = u / each;
    for (u32 i = 0; i < which; ++i) leads &= leads - 1;
    const int who = __ffs(leads) - 1;
    return {static_cast<u32>(who), u - which * each, __shfl_sync(0xffffffffu, lead.page, who),
            __shfl_sync(0xffffffffu, lead.slot, who), __shfl_sync(0xffffffffu, lead.count, who)};
}

// A chunk's keys.
template <typename T, int D, bool kWide, int kLayout>
__device__ __forceinline__ void append_keys(const RotaryArgs& r, u32 block, float* shared)
{
    const AppendArgs& a = r.a;
    const u32 lane = threadIdx.x & 31u, pairs = r.pairs, chunk = block / r.key_spread;
    const u32 base = chunk * a.chunk;
    const Lead lead = lead_of(a, chunk);
    const u32 leads = __ballot_sync(0xffffffffu, lead.leads);
    if (leads == 0) return;
    // cosines and sines of the blocks' tokens
    const u32 first = static_cast<u32>(__ffs(leads) - 1);
    const u32 tokens = __reduce_max_sync(0xffffffffu, lead.leads ? lane + lead.count : 0) - first;
    float* cosines = shared;
    float* sines = cosines + tokens * pairs;
    for (u32 i = threadIdx.x; i < tokens * pairs; i += blockDim.x) {
        const u32 token = i / pairs;
        circle_at(r, base + first + token, i - token * pairs, sines[i], cosines[i]);
    }
    __syncthreads();
    // `parts` warps to a block and head, all warps of the CTA the same number of times
    Join<D>& join = *reinterpret_cast<Join<D>*>(sines + tokens * pairs);
    const u32 total = __popc(leads) * a.c.heads, parts = a.c.block / 16, teams = kRotaryWarps / parts;
    const u32 team = (threadIdx.x >> 5) / parts, part = (threadIdx.x >> 5) - team * parts;
    for (u32 u0 = (block - chunk * r.key_spread) * teams; u0 < total; u0 += r.key_spread * teams) {
        const bool active = u0 + team < total;
        const Piece p = piece_at(lead, leads, active ? u0 + team : u0, a.c.heads);
        const u32 row = (p.who - first) * pairs, token = base + p.who;
        const Table table{cosines + row, sines + row, pairs};
        bool done = false;
        if (parts > 1 || (active && p.count > 4))
            done = append_turned<T, D, kWide, kLayout>(a, active, p.head, token, p.page, p.slot, p.count, part, parts,
                                                       table, join);
        // few tokens, for which the code for many takes longer, and elements that are not finite
        if (active && part == 0 && !done)
            append_rows<T, D, kWide, kLayout>(a, p.head, token, p.page, p.slot, p.count, table);
    }
}

// A chunk's values.
template <typename T, int D, bool kWide>
__device__ __forceinline__ void append_values(const RotaryArgs& r, u32 block)
{
    const AppendArgs& a = r.a;
    const u32 chunk = block / r.value_spread;
    const Lead lead = lead_of(a, chunk);
    const u32 leads = __ballot_sync(0xffffffffu, lead.leads), total = __popc(leads) * a.c.heads;
    for (u32 u = (block - chunk * r.value_spread) * kRotaryWarps + (threadIdx.x >> 5); u < total;
         u += r.value_spread * kRotaryWarps) {
        const Piece p = piece_at(lead, leads, u, a.c.heads);
        append_plain<T, D, kWide>(a, p.head, 1, chunk * a.chunk + p.who, p.page, p.slot, p.count);
    }
}

// 80 registers at 128 channels, of which bf16 spills 56 bytes (whole heads; f16 76); the stack frame of 40
// bytes in every form belongs to sincos.
template <typename T, int D, bool kWide, int kLayout>
__global__ void __launch_bounds__(kRotaryWarps * 32, D == 256 ? 3 : D == 128 ? 6 : 8) rotary_kernel(const RotaryArgs r)
{
    extern __shared__ float4 shared[];
    u32 block = blockIdx.x;
    if (block < r.key_blocks) {
        append_keys<T, D, kWide, kLayout>(r, block, reinterpret_cast<float*>(shared));
        return;
    }
    block -= r.key_blocks;
    if (block < r.value_blocks) {
        append_values<T, D, kWide>(r, block);
        return;
    }
    block -= r.value_blocks;
    const u64 item = static_cast<u64>(block) * kRotaryWarps + (threadIdx.x >> 5);
    const u32 token = static_cast<u32>(item / r.parts);
    const u32 part = static_cast<u32>(item - static_cast<u64>(token) * r.parts);
    if (token < r.a.tokens) turn_queries<T, D, kWide, kLayout>(r, token, part * r.part);
}

template <typename T, int D, bool kWide, int kLayout>
bool launch(const RotaryArgs& r, cudaStream_t s)
{
    const u32 join = r.a.c.block > 16 ? sizeof(Join<D>) : 0;
    const u32 smem = r.key_blocks ? (r.a.chunk - 1 + r.a.c.block) * r.pairs * 8 + join : 0;
    constexpr u32 kMost = (31 + 64) * (D / 2) * 8 + sizeof(Join<D>);
    static std::atomic<u64> seen{0};
    if (smem > 48 * 1024 && !kv_allow_smem(rotary_kernel<T, D, kWide, kLayout>, kMost, seen)) return false;
    const u64 items = static_cast<u64>(r.a.tokens) * r.parts;
    const u64 blocks = r.key_blocks + r.value_blocks + (items + kRotaryWarps - 1) / kRotaryWarps;
    return kv_launch(rotary_kernel<T, D, kWide, kLayout>, dim3(static_cast<u32>(blocks)), kRotaryWarps * 32, s, smem, 1,
                     false, r);
}

template <typename T, int D>
bool launch_wide(const RotaryArgs& r, bool neighbours, cudaStream_t s)
{
    if (!r.a.wide) return neighbours ? launch<T, D, false, kNeighbours>(r, s) : launch<T, D, false, kSplit>(r, s);
    if (neighbours) return launch<T, D, true, kNeighbours>(r, s);
    return r.pairs == D / 2 ? launch<T, D, true, kWhole>(r, s) : launch<T, D, true, kSplit>(r, s);
}

template <typename T>
bool launch_dim(const RotaryArgs& r, bool neighbours, cudaStream_t s)
{
    switch (r.a.c.dim) {
    case 64: return launch_wide<T, 64>(r, neighbours, s);
    case 128: return launch_wide<T, 128>(r, neighbours, s);
    default: return launch_wide<T, 256>(r, neighbours, s);
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
    const bool append = b->width != 0 && a.c.pages != 0;
    if (!append && x->q_heads == 0) return HBFSIM_OK;
    if (x->q_heads) {
        const u64 heads = a.c.heads, dim = a.c.dim, values = static_cast<u64>(a.c.pages) * heads * 2 * dim;
        const KvExtent out[] = {{x->q_out, u64{a.tokens} * x->q_heads * dim * 2}};
        const KvExtent in[] = {{x->q, a.tokens, x->q_stride_token, x->q_heads, x->q_stride_head, dim, 2},
                               {b->k, a.tokens, b->k_stride_token, heads, b->k_stride_head, dim, 2},
                               {b->v, a.tokens, b->v_stride_token, heads, b->v_stride_head, dim, 2},
                               {x->positions, x->axes, a.tokens, x->positions_stride},
                               {x->freq, u64{x->pairs} * 8},
                               {x->axis, x->pairs},
                               {b->table, a.seqs, a.width, b->table_stride},
                               {b->start, u64{a.seqs} * 4},
                               {b->offsets, b->offsets ? u64{a.seqs} * 4 + 4 : 0},
                               {a.c.data, values * a.c.block},
                               {a.c.bounds, values},
                               {a.c.scale, values / dim * 4}};
        if (kv_would_race(out, in, {-1})) return HBFSIM_INVALID_ARGUMENT;
    }
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
    // Chunks as in kv_append.cu; few tokens get a warp to each head and side.  Large batches in blocks of
    // 16 get chunks of 32 tokens: what comes before the first row of a chunk (the search for its blocks,
    // the cosines) is shared by two blocks (prompts of 31,668 tokens: 139 us with 16, 134 us with 32; in
    // blocks of 32, 141 and 160 us, of 64, 173 and 207 us).
    const u32 heads = a.c.heads, groups = (r.q_heads + kRotaryHeads - 1) / kRotaryHeads;
    const u64 warps = static_cast<u64>(kv_sm_count()) * 16;  // resident at once
    a.chunk = 1;
    const u32 most = a.c.block == 16 ? 32 : 16;
    while (a.chunk < most && static_cast<u64>(a.tokens) * heads * 2 > a.chunk * warps) a.chunk *= 2;
    if (append) {
        // A CTA takes as many heads' keys of a block at once as it has warps for, 16 rows to a warp; where
        // that makes many more CTAs than are resident, eight share a block's cosines, one after the other
        // (those prompts in blocks of 16: 145 us by four, 134 us by eight; of 32: 176 by two, 141 by eight;
        // of 64: 259 by one, 206 by two, 178 by four, 173 by eight).
        const u32 chunks = (a.tokens + a.chunk - 1) / a.chunk, teams = kRotaryWarps / (a.c.block / 16);
        const u64 pieces = (static_cast<u64>(a.tokens) / a.c.block + a.seqs) * heads;
        const u32 by = pieces > 12ull * teams * kv_sm_count() ? 8 : teams;
        r.key_spread = (heads + by - 1) / by;
        r.value_spread = (heads + kRotaryWarps - 1) / kRotaryWarps;
        r.key_blocks = chunks * r.key_spread;
        r.value_blocks = chunks * r.value_spread;
    }
    // A token's queries: all heads to a warp that are not needed to fill the device.
    r.part = static_cast<u32>(std::max<u64>(1, std::min<u64>(groups, static_cast<u64>(a.tokens) * groups / warps)));
    r.parts = (groups + r.part - 1) / r.part;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool ok = b->type == HBFSIM_KV_BF16 ? launch_dim<__nv_bfloat16>(r, x->neighbours != 0, s)
                                              : launch_dim<__half>(r, x->neighbours != 0, s);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
