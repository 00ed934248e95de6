// kv_attention.cu -- attention of the newest tokens over the 8-bit paged
// cache (kv_v1.h), over all blocks of a sequence or over listed ones.
//
// The query rows that share a key/value head (group heads times tokens) are
// taken 8 to 24 at a time as the narrow side of the tensor-core products, so
// that the tokens are the wide one:
//
//   S^T [16 tokens x rows]  = K [16 x D] Q^T [D x rows]
//   O^T [D x rows]         += V^T [D x 16 tokens] P^T [16 x rows]
//
// K and V are read in their natural order straight into the fragments of
// mma.m16n8k16: the order of the channels inside a dot product and of the
// tokens inside a sum is free, so each lane takes 16 contiguous bytes.  e4m3
// widens to f16 without loss.  A block's scales are powers of two: the keys'
// is applied in fp32 to the scores, the values' to the probabilities, relative
// to a reference of the row.  Queries are scaled per row by a power of two
// into f16's range, which keeps all that is within 2^29 of the row's largest.
// Scores, the running maximum, sums and the output accumulate in fp32.  The
// probabilities, times the value scale, are rounded to f16 for the second
// product only: 2^-11 relative, no more than the output type's own rounding,
// down to 2^-24 of the row's largest (2^-14 where the scales differ by
// kNear); what is smaller loses 2^-35 (2^-25) of the largest.  Where scales
// differ by more, the product takes bf16 pairs (2^-17 relative).  The sums and
// the block weights use the probabilities unrounded.
//
// Work: the 16-token tiles of all segments (sequence, head, row tile; for
// lists also the token) form one line that is cut into equal shares, one per
// resident CTA, so that ragged lengths leave no SM idle.  A CTA's 4 warps
// stride over the tiles of its share of a segment, each with a ring of
// asynchronous copies of its own (no block barrier inside the loop), join
// through shared memory and leave one partial result per segment met;
// finish_kernel joins the partials of a segment and turns the tiles' sums
// into block weights.  Short segments have a CTA each, of 8 warps if it has an
// SM to itself, and need neither (one of 301 tokens takes 7.0 us); few that
// are longer have a team of CTAs each.
//
// One decode step of 64 sequences of 1024 to 32768 tokens, 8 heads of 128
// channels with 4 rows each, takes 402 us with weights: 2.21 GB at 5.5 TB/s,
// 85 % of a copy's rate, DRAM's bound; 12 warps an SM take 43 % of the issue
// slots, 282 instructions for the 4 KB of a tile.  128 listed blocks per head
// take 64 us (272 MB at 4.2 TB/s): shares of 150 tiles begin and join more
// often.  One sequence of 262,147 tokens takes 105 us (539 MB at 5.1 TB/s).
// 40 rows on 8 sequences of 700 to 9001 tokens take 64 us, three passes that
// are bound by the latency of their instructions (46 % of the slots).
#include "kv.h"
#include "kv_plan.h"

#include <algorithm>
#include <type_traits>

namespace hbfb {
namespace {

// The probabilities of a row stand against a reference of its scores (log2), which moves up only when
// a score is 2^kAbove above it: a tile then costs a vote instead of a maximum over the lanes.  After a
// move the largest is 2^kPlace, which f16 holds exactly (it may be nearly all of the row), and f16
// keeps its 11 bits down to 2^-24 of it.  For the product with the values they are multiplied by
// their block's value scale over the greatest that the warp has met.
constexpr float kAbove = 15.0f, kPlace = 10.0f;
// That holds for scales within kNear of each other.  Past it a block of large scale and no weight
// would push the others out of f16's range, so from there on the warp keeps a second reference for
// each row, of scores plus the logarithm of their value scale, a whole number that only what really
// counts moves up, and
// takes pairs of bf16 (16 bits, fp32's range) in twice the products.  They lie 2^kLift higher: up to
// 2^kFarAbove, which times 448 times 2^31 tokens is still a number, and down to 2^-126, so that not
// even values that are all 0 in a block of large scale and weight hide the others.  With every other
// block 2^40 below its neighbours the decode step takes 457 us instead of 402, 40 rows 92 instead of
// 64; all in pairs from the start would cost every call that.
constexpr float kNear = 1024.0f;
constexpr float kFarAbove = 85.0f, kFarPlace = 81.0f, kLift = 70.0f;
constexpr float kNoScore = -3.0e38f;  // reference of a row without a score
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr u32 kFinishThreads = 256; // blocks per CTA of finish_kernel

struct AttentionArgs {
    KvView c;
    KvQuery q;
    float scale2;          // softmax scale times log2(e)
    u32 top;               // lists; 0: every block
    const int* blocks;
    const int* counts;
    void* out;
    float* lse;
    float* weights;
    // segments: ((seq * lists + t) * heads + h) * row_tiles + rt, lists = tokens or 1;
    // `units` runs of `per_unit` neighbouring segments have equally many tiles
    u32 lists, row_tiles, rows;   // rows of one (sequence, list, head)
    u32 units, per_unit;
    u32 workers;                  // CTAs of attention_kernel
    u32 team;                     // CTAs (a cluster) that finish a segment together
    u32 tiles;                    // 16-token tiles per segment at most
    float* part_o;                // [workers + segments][8 NT][D], at worker + segment, channels
                                  // in the joined order
    float2* part_ml;              // [workers + segments][8 NT]: reference of the scores, sum
    float* part_ref;              // [workers + segments][8 NT]: reference of the values
    uint2* span;                  // [segments]: first and last worker (segments with tiles)
    float2* tile_sums;            // [segments][tiles][8 NT] or NULL: sum of exponentials, reference
};

// Four stored values as f16 pairs: exact.
__device__ __forceinline__ void e4m3x4_to_f16(u32 four, u32& lo, u32& hi)
{
    asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

__device__ __forceinline__ void mma16816(float (&d)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0,
                                         u32 b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ u32 transpose8x8(u32 x)
{
    u32 r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ u32 pack_f16(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const u32*>(&h);
}

__device__ __forceinline__ u32 times(u32 pair, __half2 by)
{
    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&pair), by);
    return *reinterpret_cast<const u32*>(&y);
}

__device__ __forceinline__ void mma16816_bf16(float (&d)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0,
                                              u32 b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ u32 pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const u32*>(&h);
}

// Stored values from f16 to bf16: exact (4 significant bits, 2^-9 to 448).
__device__ __forceinline__ u32 bf16_of(u32 pair)
{
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    return pack_bf16(y.x, y.y);
}

// What two bf16 roundings leave of a pair.
__device__ __forceinline__ u32 rest_of(u32 pair, float lo, float hi)
{
    return pack_bf16(lo - __uint_as_float(pair << 16), hi - __uint_as_float(pair & 0xffff0000u));
}

__device__ __forceinline__ float exp2_fast(float x)  // 2^-22 relative, 0 for -inf
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 1 / x for a power of two x, 2^-126 <= x <= 2^126: exact.
__device__ __forceinline__ float inverse_power(float x)
{
    return __int_as_float((254 << 23) - __float_as_int(x));
}

// Exponent of a power of two.
__device__ __forceinline__ float exponent_of(float x) { return static_cast<float>((__float_as_int(x) >> 23 & 0xff) - 127); }

// x * 2^by in two steps: the power may be past fp32's range where the result is not.
__device__ __forceinline__ float at_power(float x, float by)
{
    const float half = rintf(0.5f * by);
    return x * exp2_fast(half) * exp2_fast(by - half);
}

// Place of byte o of a tile side in shared memory: the 16-byte pieces of a
// 128-byte line are exchanged by the line's number, so that the lanes that
// read one channel range of 4 tokens, or 8 tokens of one range, meet
// different banks.
__device__ __forceinline__ u32 swizzle(u32 o) { return o ^ ((o >> 3) & 0x70u); }

struct Segment {
    u32 seq, t, h, rt, index;
    int length;      // tokens of the sequence
    u32 tiles;       // 16-token tiles of this segment
};

// 16-token tiles of each segment of a unit (a sequence, or one list).
__device__ __forceinline__ u32 unit_tiles(const AttentionArgs& a, u32 unit)
{
    if (a.blocks)
        return static_cast<u32>(min(max(a.counts[unit], 0), static_cast<int>(a.top))) *
               (a.c.block / 16);
    return (static_cast<u32>(kv_length(a.q.lengths, unit, a.q.width, a.c.block)) + 15) / 16;
}

__device__ __forceinline__ Segment segment_of(const AttentionArgs& a, u32 index)
{
    Segment s;
    s.index = index;
    s.rt = index % a.row_tiles;
    u32 r = index / a.row_tiles;
    s.h = r % a.c.heads;
    r /= a.c.heads;
    s.t = r % a.lists;
    s.seq = r / a.lists;
    s.length = kv_length(a.q.lengths, s.seq, a.q.width, a.c.block);
    s.tiles = unit_tiles(a, index / a.per_unit);
    return s;
}

// Tiles per share of a line of `total` tiles.
__device__ __forceinline__ u64 share_of(const AttentionArgs& a, u64 total)
{
    const u64 even = (total + a.workers - 1) / a.workers;
    return even > kShare ? even : kShare;
}

// Where this CTA's share of the line of all tiles begins and ends, the unit
// that holds its beginning and where that unit begins.  Each thread has a run
// of units; a scan over the block gives their places.
struct Place {
    u64 at, stop, begin;
    u32 unit;
};

__device__ __forceinline__ Place place_of(const AttentionArgs& a, u64* sums, Place* found)
{
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const u32 each = (a.units + kWarps * 32 - 1) / (kWarps * 32);
    const u32 from = min(threadIdx.x * each, a.units), to = min(from + each, a.units);
    u64 mine = 0;
#pragma unroll 4
    for (u32 u = from; u < to; ++u) mine += static_cast<u64>(unit_tiles(a, u)) * a.per_unit;
    u64 upto = mine;
#pragma unroll
    for (u32 o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (u32 w = 0; w < kWarps; ++w) {
        if (w < warp) upto += sums[w];
        total += sums[w];
    }
    const u64 share = share_of(a, total), at = blockIdx.x * share;
    if (threadIdx.x == 0 && at >= total) found->at = found->stop = 0;
    if (at < total && at >= upto - mine && at < upto) {
        Place p{at, min(at + share, total), upto - mine, from};
        for (;; ++p.unit) {
            const u64 n = static_cast<u64>(unit_tiles(a, p.unit)) * a.per_unit;
            if (at < p.begin + n) break;
            p.begin += n;
        }
        *found = p;
    }
    __syncthreads();
    return *found;
}

// Position of the query token behind a row of the segment (-1: sees nothing).
__device__ __forceinline__ int row_position(const AttentionArgs& a, const Segment& s, u32 row)
{
    const u32 t = a.blocks ? s.t : row / a.q.group;
    return max(s.length - static_cast<int>(a.q.tokens) + static_cast<int>(t), -1);
}

// Joined values lie as the lanes hold them: channel g D/8 + 2k + e of a row at
// 16 k + 2 g + e, so that lanes that write or read together meet different
// banks.  The channel at a place:
__device__ __forceinline__ u32 channel_of(u32 dim, u32 at) { return at % 16 / 2 * (dim / 8) + at / 16 * 2 + at % 2; }

// Row of out and lse behind a row of the segment.
__device__ __forceinline__ u64 out_row(const AttentionArgs& a, const Segment& s, u32 row)
{
    const u32 t = a.blocks ? s.t : row / a.q.group;
    return (static_cast<u64>(s.seq) * a.q.tokens + t) * a.q.q_heads + s.h * a.q.group + row % a.q.group;
}

__device__ __forceinline__ void put_out(const AttentionArgs& a, const Segment& s, u32 row, u32 d, float y)
{
    const u64 at = out_row(a, s, row) * a.c.dim + d;
    if (a.q.type == HBFSIM_KV_BF16) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    else static_cast<__half*>(a.out)[at] = __float2half_rn(y);
}

// Depth of a warp's ring.
template <int D>
constexpr u32 kStages = D == 256 ? 3 : 4;
// One row tile's queries stay in registers; more are read from shared memory for each tile.
template <int D, int NT>
constexpr bool kSharedQueries = NT > 1 || D == 256;
// Shared memory: rings (later the joined values), notes, sums, queries, row factors and ends, a word.
template <int D, int NT, u32 W>  // W warps
struct Layout {
    static constexpr u32 ring = W * kStages<D> * 32 * D;
    static constexpr u32 join = W * 8 * NT * (D + 8) * 4;
    static constexpr u32 notes = ring > join ? ring : join;
    static constexpr u32 join_ml = notes + W * kStages<D> * 16;
    static constexpr u32 join_ref = join_ml + W * 8 * NT * 8;
    static constexpr u32 join_factor = join_ref + W * 8 * NT * 4;
    static constexpr u32 row_power = join_factor + W * 8 * NT * 8;
    static constexpr u32 queries = row_power + 8 * NT * 8;
    static constexpr u32 factors = queries + (kSharedQueries<D, NT> ? NT * D * 16 : 0);
    static constexpr u32 ends = factors + 8 * NT * 4;
    static constexpr u32 line = ends + 8 * NT * 4;  // of the split; for whole segments:
    static constexpr u32 whole_sums = line;         // [tiles][8 NT], if there are weights
    static constexpr u32 bytes = line + 8 * W + sizeof(u64) * 4;
    static constexpr u32 most = whole_sums + whole_tiles(NT, W) * 8 * NT * 8;
};

// One segment's tiles [first, end) by one CTA; the partial result goes to `part` (a whole segment:
// joined with those of its team, in which this CTA is number `part`).
template <int D, int NT, bool kWhole, u32 W>
__device__ __forceinline__ void run_segment(const AttentionArgs& a, const Segment& seg, u32 first,
                                            u32 end, u64 part, u8* smem)
{
    constexpr int R = 8 * NT;
    constexpr int KC = D / 64;      // 16-byte pieces of a key row per lane
    constexpr int VW = D / 32;      // 4-byte words of a value row per lane
    constexpr u32 NS = kStages<D>;
    constexpr u32 kSide = 16 * D;   // bytes of a tile's keys, and of its values
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3u;
    u8* ring = smem + warp * NS * 2 * kSide;
    // after the loop [W][R][D + 8], channels in the joined order
    float* join_o = reinterpret_cast<float*>(smem);
    using L = Layout<D, NT, W>;
    constexpr bool kShared = kSharedQueries<D, NT>;
    int4* note = reinterpret_cast<int4*>(smem + L::notes) + warp * NS;  // position, -, scales
    float2* join_ml = reinterpret_cast<float2*>(smem + L::join_ml);     // [W][R]
    float* join_ref = reinterpret_cast<float*>(smem + L::join_ref);     // [W][R]
    float2* join_factor = reinterpret_cast<float2*>(smem + L::join_factor);  // [W][R]
    float2* row_power = reinterpret_cast<float2*>(smem + L::row_power);      // [R]
    uint4* queries = reinterpret_cast<uint4*>(smem + L::queries);       // [NT][D / 32][32 lanes]
    float* factors = reinterpret_cast<float*>(smem + L::factors);       // [R]
    int* ends = reinterpret_cast<int*>(smem + L::ends);                 // [R]: last position a row sees
    const u32 ring_at = static_cast<u32>(__cvta_generic_to_shared(ring));
    const u32 note_at = static_cast<u32>(__cvta_generic_to_shared(note));
    const u32 rows = min(static_cast<u32>(R), a.rows - seg.rt * R);
    const u32 block = a.c.block, sub_bits = 27 - __clz(block);  // tiles of a block: 1 << sub_bits

    const int sees_least = row_position(a, seg, seg.rt * R);
    const int sees_most = row_position(a, seg, seg.rt * R + rows - 1);
    const int* table = a.q.table + static_cast<i64>(seg.seq) * a.q.table_stride;
    const int* list = a.blocks ? a.blocks + ((static_cast<u64>(seg.seq) * a.lists + seg.t) *
                                                 a.c.heads + seg.h) * a.top
                               : nullptr;
    const u32 have = (static_cast<u32>(seg.length) + block - 1) / block;
    const u32 turns = first + warp < end ? (end - first - warp + W - 1) / W : 0;

    const u32 page_bytes = a.c.heads * 2 * block * D, page_scales = a.c.heads * 2;
    const u8* head_data = a.c.data + seg.h * 2 * block * D + lane * 16;
    const float* head_scale = a.c.scale + seg.h * 2;
    // Copies of the warp's i-th tile into a stage (i % NS).  The blocks and pages of 32 turns are
    // looked up at once, one per lane.
    int my_page = -1;
    u32 my_block = 0;
    auto issue = [&](u32 i, u32 stage) {
        if (i < turns) {
            if (i % 32 == 0) {
                my_page = -1;
                if (i + lane < turns) {
                    my_block = (first + warp + (i + lane) * W) >> sub_bits;
                    if (list) my_block = static_cast<u32>(list[my_block]);
                    if (my_block < have) my_page = kv_page(table, my_block, a.c.pages);
                }
            }
            const int page = __shfl_sync(0xffffffffu, my_page, i % 32);
            const u32 j = __shfl_sync(0xffffffffu, my_block, i % 32);
            const u32 sub = (first + warp + i * W) & ((1u << sub_bits) - 1u);
            const int p0 = static_cast<int>(j * block + sub * 16);
            const bool there = page >= 0 && p0 <= sees_most;
            if (lane == 0) note[stage].x = there ? p0 : -1;
            if (there) {
                const u8* from = head_data + static_cast<u64>(page) * page_bytes + sub * (16 * D);
                const u8* from_v = from + block * D;
                // swizzle(k + lane * 16) for k a multiple of 512: the line number's third bit is k's
                const u32 to = ring_at + stage * 2 * kSide;
                const u32 even = to + swizzle(lane * 16), odd = to + swizzle(512 + lane * 16);
#pragma unroll
                for (u32 k = 0; k < kSide; k += 1024) {
                    kv_copy16(even + k, from + k);
                    kv_copy16(odd + k, from + k + 512);
                }
#pragma unroll
                for (u32 k = 0; k < kSide; k += 1024) {
                    kv_copy16(even + kSide + k, from_v + k);
                    kv_copy16(odd + kSide + k, from_v + k + 512);
                }
                if (lane == 0) kv_copy8(note_at + stage * 16 + 8, head_scale + static_cast<u64>(page) * page_scales);
            }
        }
        kv_copy_commit();
    };
#pragma unroll
    for (u32 i = 0; i + 1 < NS; ++i) issue(i, i);

    // Queries: row n = 8 nt + g, scaled by a power of two so that the largest is in
    // [2^14, 2^15); its factor is scale2 over that power.
    u32 qf[kShared ? 1 : D / 16][2];
    float factor0 = 0.0f, factor1 = 0.0f;  // of the columns 2c, 2c + 1
    for (u32 nt = kShared ? warp : 0; nt < NT; nt += kShared ? W : 1) {
        const u32 n = nt * 8 + g;
        float x[KC][16];
        float most = 0.0f;
        if (n < rows) {
            const u32 row = seg.rt * R + n;
            const u32 t = a.blocks ? seg.t : row / a.q.group;
            const u32 qh = seg.h * a.q.group + row % a.q.group;
            const i64 at = static_cast<i64>(seg.seq) * a.q.stride_seq +
                           static_cast<i64>(t) * a.q.stride_token +
                           static_cast<i64>(qh) * a.q.stride_head;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                kv_load<16>(a.q.q, at + (c * KC + k) * 16, a.q.type, a.q.wide, x[k]);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (fabsf(x[k][i]) <= 3.402823466e38f) most = fmaxf(most, fabsf(x[k][i]));
            }
        } else {
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[k][i] = 0.0f;
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        int e = 15;
        if (most > 0.0f) frexpf(most, &e);
        e = max(15 - e, -126);
        e = min(e, 126);
        const float up = kv_power(e);
        const float f = a.scale2 * kv_power(-e);
        if constexpr (kShared) {
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int w = 0; w < 4; w += 2)
                    queries[(nt * (D / 32) + k * 2 + w / 2) * 32 + lane] =
                        make_uint4(pack_f16(x[k][4 * w] * up, x[k][4 * w + 1] * up),
                                   pack_f16(x[k][4 * w + 2] * up, x[k][4 * w + 3] * up),
                                   pack_f16(x[k][4 * w + 4] * up, x[k][4 * w + 5] * up),
                                   pack_f16(x[k][4 * w + 6] * up, x[k][4 * w + 7] * up));
            if (c == 0) factors[n] = f;
        } else {
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    qf[k * 4 + w][0] = pack_f16(x[k][4 * w] * up, x[k][4 * w + 1] * up);
                    qf[k * 4 + w][1] = pack_f16(x[k][4 * w + 2] * up, x[k][4 * w + 3] * up);
                }
            factor0 = __shfl_sync(0xffffffffu, f, 8 * c);
            factor1 = __shfl_sync(0xffffffffu, f, 8 * c + 4);
        }
    }
    if (threadIdx.x < R)
        ends[threadIdx.x] = row_position(a, seg, seg.rt * R + min(static_cast<u32>(threadIdx.x), rows - 1));
    __syncthreads();

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2], ref[NT][2];  // reference and sum of the scores; of the values, if far
    float value_scale = 0.0f, least_scale = INFINITY;  // the greatest and the least value scale met
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[nt][i][k] = 0.0f;
        m[nt][0] = m[nt][1] = ref[nt][0] = ref[nt][1] = kNoScore;
        l[nt][0] = l[nt][1] = 0.0f;
    }
    // where the lane's pieces lie in a tile side, and the same 8 tokens further: at D = 64 that
    // is 4 lines on, which turns the exchange by 4
    auto further = [](u32 at) { return D == 64 ? (at ^ 0x40u) + 512u : at + 8u * D; };
    u32 key_at[KC], value_at[2][VW >= 4 ? VW / 4 : 1];
#pragma unroll
    for (int k = 0; k < KC; ++k) key_at[k] = swizzle(g * D + (c * KC + k) * 16);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int w = 0; w < (VW >= 4 ? VW / 4 : 1); ++w)
            value_at[x][w] = kSide + swizzle((2 * c + x) * D + g * (D / 8) + w * 16);

    // Mask of the f16 halves that are numbers, and the first token (0..15) of a row of the value
    // fragment, over the 4 lanes that hold it, that is none (a large number without one).
    auto numbers = [](u32 x) {
        const __half2 y = *reinterpret_cast<const __half2*>(&x);
        return __heq2_mask(y, y);
    };
    auto first_nan = [&](u32 lo, u32 hi) {
        int t = !(lo & 0xffffu) ? 0 : !(lo >> 16) ? 1 : !(hi & 0xffffu) ? 8 : !(hi >> 16) ? 9 : 1 << 20;
        t += static_cast<int>(2 * c);
        t = min(t, __shfl_xor_sync(0xffffffffu, t, 1));
        return min(t, __shfl_xor_sync(0xffffffffu, t, 2));
    };
    auto multiply = [&](float by) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[nt][k][x] *= by;
    };
    // One tile.  `edge`: some row does not see all of its tokens; `far`: see kNear.  False, with
    // nothing summed, where this tile's value scale is the first that is far from those before it.
    auto consume = [&](auto is_edge, auto is_far, const u8* tile, int p0, float key_scale, float new_scale,
                       float2* tile_out) -> bool {
        constexpr bool kEdge = decltype(is_edge)::value, kFar = decltype(is_far)::value;
        // with one row tile two sums, so that products need not wait for each other
        constexpr int kSums = NT == 1 ? 2 : 1;
        float s[NT][kSums][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < kSums; ++x)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[nt][x][k] = 0.0f;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const uint4 k0 = *reinterpret_cast<const uint4*>(tile + key_at[k]);
            const uint4 k1 = *reinterpret_cast<const uint4*>(tile + further(key_at[k]));
            const u32 w0[4] = {k0.x, k0.y, k0.z, k0.w};
            const u32 w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
            for (int w = 0; w < 4; w += 2) {
                u32 x[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    e4m3x4_to_f16(w0[w + i], x[i][0], x[i][2]);
                    e4m3x4_to_f16(w1[w + i], x[i][1], x[i][3]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint4 q;
                    if constexpr (kShared) q = queries[(nt * (D / 32) + k * 2 + w / 2) * 32 + lane];
                    else q = make_uint4(qf[k * 4 + w][0], qf[k * 4 + w][1], qf[k * 4 + w + 1][0], qf[k * 4 + w + 1][1]);
                    mma16816(s[nt][0], x[0][0], x[0][1], x[0][2], x[0][3], q.x, q.y);
                    mma16816(s[nt][kSums - 1], x[1][0], x[1][1], x[1][2], x[1][3], q.z, q.w);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if constexpr (kSums == 2) s[nt][0][k] += s[nt][1][k];
        u32 v[4][VW];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if constexpr (VW == 2) {
                const uint2 y = *reinterpret_cast<const uint2*>(
                    tile + (x >> 1 ? further(value_at[x & 1][0]) : value_at[x & 1][0]));
                v[x][0] = y.x;
                v[x][1] = y.y;
            } else {
#pragma unroll
                for (int w = 0; w < VW; w += 4) {
                    const u32 at = value_at[x & 1][w / 4];
                    const uint4 y = *reinterpret_cast<const uint4*>(tile + (x >> 1 ? further(at) : at));
                    v[x][w] = y.x;
                    v[x][w + 1] = y.y;
                    v[x][w + 2] = y.z;
                    v[x][w + 3] = y.w;
                }
            }
        }
        if constexpr (!kFar) {
            least_scale = fminf(least_scale, new_scale);
            if (new_scale > value_scale || new_scale * kNear < value_scale) {
                if (value_scale > 0.0f && fmaxf(new_scale, value_scale) > least_scale * kNear) return false;
                multiply(value_scale * inverse_power(new_scale));  // a change rescales what is summed
                value_scale = new_scale;
            }
        }
        const float value_log2 = exponent_of(new_scale);
        const __half2 relative = __float2half2_rn(new_scale * inverse_power(value_scale));
        u32 b[NT][2], b_rest[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float p[4], w[4], sum[2];  // scores against the references, then probabilities and factors
            float2 factor = make_float2(factor0, factor1);
            if constexpr (kShared) factor = *reinterpret_cast<const float2*>(factors + nt * 8 + 2 * c);
            const float scaled[2] = {factor.x * key_scale, factor.y * key_scale};
            auto against = [&]() {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    p[i] = fmaf(s[nt][0][i], scaled[i], -m[nt][i]);
                    p[2 + i] = fmaf(s[nt][0][2 + i], scaled[i], -m[nt][i]);
                    if constexpr (kFar) {
                        const float at = value_log2 - ref[nt][i];  // exact: whole numbers
                        w[i] = fmaf(s[nt][0][i], scaled[i], at);
                        w[2 + i] = fmaf(s[nt][0][2 + i], scaled[i], at);
                    }
                    if constexpr (kEdge) {
                        const int end = ends[nt * 8 + 2 * c + i];
                        if (p0 + static_cast<int>(g) > end) p[i] = w[i] = -INFINITY;
                        if (p0 + static_cast<int>(g) + 8 > end) p[2 + i] = w[2 + i] = -INFINITY;
                    }
                }
            };
            against();
            bool moves = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])) > kAbove;
            if constexpr (kFar) moves |= fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])) > kFarAbove;
            if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float most = -INFINITY;
                    if (p[i] > -INFINITY) most = s[nt][0][i] * scaled[i];
                    if (p[2 + i] > -INFINITY) most = fmaxf(most, s[nt][0][2 + i] * scaled[i]);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1)
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                    const float now = fmaxf(m[nt][i], most - kPlace);
                    const float shrink = exp2_fast(m[nt][i] - now);
                    l[nt][i] *= shrink;
                    m[nt][i] = now;
                    float once = shrink, again = 1.0f;
                    if constexpr (kFar) {
                        const float now_ref = fmaxf(ref[nt][i], ceilf(most + value_log2) - kFarPlace);
                        const float by = ref[nt][i] - now_ref, half = rintf(0.5f * by);  // as at_power
                        once = exp2_fast(half);
                        again = exp2_fast(by - half);
                        ref[nt][i] = now_ref;
                    }
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        o[nt][k][i] *= once;
                        o[nt][k][2 + i] *= once;
                        if constexpr (kFar) {
                            o[nt][k][i] *= again;
                            o[nt][k][2 + i] *= again;
                        }
                    }
                }
                against();
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[i] = exp2_fast(p[i]);
                p[2 + i] = exp2_fast(p[2 + i]);
                sum[i] = p[i] + p[2 + i];
                l[nt][i] += sum[i];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (kFar) {
                    const float x = exp2_fast(w[2 * i]), y = exp2_fast(w[2 * i + 1]);
                    const u32 most = pack_bf16(x, y);
                    b[nt][i] = transpose8x8(most);
                    b_rest[nt][i] = transpose8x8(rest_of(most, x, y));
                } else {
                    b[nt][i] = transpose8x8(times(pack_f16(p[2 * i], p[2 * i + 1]), relative));
                }
            }
            if (tile_out) {
                // the two columns' sums over the lanes of all g, the even g keeping the first
                const float mine = g & 1 ? sum[1] : sum[0], other = g & 1 ? sum[0] : sum[1];
                float all = mine + __shfl_xor_sync(0xffffffffu, other, 4);
                all += __shfl_xor_sync(0xffffffffu, all, 8);
                all += __shfl_xor_sync(0xffffffffu, all, 16);
                const u32 row = nt * 8 + 2 * c + g;
                if (g < 2 && row < rows) tile_out[row] = make_float2(all, g ? m[nt][1] : m[nt][0]);
            }
        }
        u32 keep_lo = 0xffffffffu, keep_hi = 0xffffffffu;  // value tokens that some row sees
        bool staggered = false;
        if constexpr (kEdge) {
            const int n = sees_most - p0 - static_cast<int>(2 * c);  // token 2c + i is seen if i <= n
            keep_lo = (n >= 0 ? 0x0000ffffu : 0u) | (n >= 1 ? 0xffff0000u : 0u);
            keep_hi = (n >= 8 ? 0x0000ffffu : 0u) | (n >= 9 ? 0xffff0000u : 0u);
            staggered = sees_least < sees_most;
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const u32 pick = half ? 0x7362 : 0x5140;
                const u32 lo = __byte_perm(v[0][w], v[1][w], pick), hi = __byte_perm(v[2][w], v[3][w], pick);
                u32 a0, a1, a2, a3;
                e4m3x4_to_f16(lo, a0, a1);
                e4m3x4_to_f16(hi, a2, a3);
                const int k = w * 2 + half;
                if constexpr (kEdge) {
                    a0 &= keep_lo;
                    a1 &= keep_lo;
                    a2 &= keep_hi;
                    a3 &= keep_hi;
                    if (staggered) {
                        // Rows end at different tokens: a NaN past a row's end must not meet the
                        // row, so NaN goes in as 0 and then to the rows that see it.
                        const u32 n0 = numbers(a0), n1 = numbers(a1), n2 = numbers(a2), n3 = numbers(a3);
                        if (__any_sync(0xffffffffu, (n0 & n1 & n2 & n3) != 0xffffffffu)) {
                            a0 &= n0;
                            a1 &= n1;
                            a2 &= n2;
                            a3 &= n3;
                            const int t0 = p0 + first_nan(n0, n2), t1 = p0 + first_nan(n1, n3);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const int end = ends[nt * 8 + 2 * c + i];
                                    if (end >= t0) o[nt][k][i] = __int_as_float(0x7fffffff);
                                    if (end >= t1) o[nt][k][2 + i] = __int_as_float(0x7fffffff);
                                }
                        }
                    }
                }
                if constexpr (kFar) {
                    a0 = bf16_of(a0), a1 = bf16_of(a1), a2 = bf16_of(a2), a3 = bf16_of(a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816_bf16(o[nt][k], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                        mma16816_bf16(o[nt][k], a0, a1, a2, a3, b_rest[nt][0], b_rest[nt][1]);
                    }
                } else {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16816(o[nt][k], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                }
            }
        }
        return true;
    };

    u32 stage = 0;
    float2* whole_sums = reinterpret_cast<float2*>(smem + L::whole_sums);
    float2* tile_out = nullptr;
    if (a.weights)
        tile_out = (kWhole ? whole_sums : a.tile_sums + (static_cast<u64>(seg.index) * a.tiles + first) * R) + warp * R;
    auto nothing = [&]() {
        if (tile_out && lane < rows) tile_out[lane] = make_float2(0.0f, kNoScore);
    };
    u32 i = 0;
    auto next = [&]() {
        stage = stage + 1 == NS ? 0 : stage + 1;
        if (tile_out) tile_out += W * R;
        ++i;
    };
    auto wait = [&]() {
        kv_copy_wait<NS - 2>();
        __syncwarp();  // the stage is there, and every lane is done with the one before it
        issue(i + NS - 1, stage == 0 ? NS - 1 : stage - 1);
    };
    for (; i < turns; next()) {
        wait();
        const int4 noted = note[stage];
        const u8* tile = ring + stage * 2 * kSide;
        const float key_scale = __int_as_float(noted.z), new_scale = __int_as_float(noted.w);
        bool done = true;
        if (noted.x < 0) nothing();
        else if (noted.x + 15 > sees_least)
            done = consume(std::true_type{}, std::false_type{}, tile, noted.x, key_scale, new_scale, tile_out);
        else
            done = consume(std::false_type{}, std::false_type{}, tile, noted.x, key_scale, new_scale, tile_out);
        if (!done) break;
    }
    // the references of the rows' values, whole numbers from here on, lifted
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const float up = ceilf(m[nt][x]), by = exp2_fast(m[nt][x] - up + kLift);
            ref[nt][x] = up + (exponent_of(value_scale) - kLift);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                o[nt][k][x] *= by;
                o[nt][k][2 + x] *= by;
            }
        }
    for (bool waited = true; i < turns; next(), waited = false) {
        if (!waited) wait();
        const int4 noted = note[stage];
        if (noted.x < 0) nothing();
        else
            consume(std::true_type{}, std::true_type{}, ring + stage * 2 * kSide, noted.x, __int_as_float(noted.z),
                    __int_as_float(noted.w), tile_out);
    }
    kv_copy_wait<0>();
    __syncthreads();  // every ring is at rest: its memory takes the joined values
    // join the warps: every warp's sums and values at its own references
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float sum = l[nt][i];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            const u32 row = nt * 8 + 2 * c + i;
            if (g == 0) {
                join_ml[warp * R + row] = make_float2(m[nt][i] == kNoScore ? -INFINITY : m[nt][i], sum);
                join_ref[warp * R + row] = ref[nt][i];
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                *reinterpret_cast<float2*>(join_o + (warp * R + row) * (D + 8) + k * 16 + g * 2) =
                    make_float2(o[nt][k][i], o[nt][k][2 + i]);
        }
    __syncthreads();
    float* inverses = reinterpret_cast<float*>(ends);
    // what a team's CTA joins lies behind its warps' values, in what was the ring
    const u32 team = kWhole && W > kWarps ? a.team : 1u, rank = kWhole ? static_cast<u32>(part) : 0u;
    float* cta_o = reinterpret_cast<float*>(smem + L::join);     // [R][D]
    float2* cta_ml = reinterpret_cast<float2*>(smem + L::notes); // [R]
    float* cta_ref = reinterpret_cast<float*>(cta_ml + R);       // [R]
    static_assert(W == kWarps || (L::join + R * D * 4 <= L::ring && NS * W * 16 >= R * 12));
    auto peek = [](const float* mine, u32 r) { return __uint_as_float(kv_peek(reinterpret_cast<const u32*>(mine), r)); };
    auto peek2 = [](const float2* mine, u32 r) {
        const u64 x = kv_peek(reinterpret_cast<const u64*>(mine), r);
        return make_float2(__uint_as_float(static_cast<u32>(x)), __uint_as_float(static_cast<u32>(x >> 32)));
    };
    // a thread for each row and warp: the powers of two that the warp's values are multiplied by, in
    // two steps as at_power takes them; the first warp's also finish the row's sum
    auto steps = [](float by) {
        const float half = rintf(0.5f * by);
        return make_float2(exp2_fast(half), exp2_fast(by - half));
    };
    // what the output of a whole segment's row and the weights of its blocks need
    auto finish_row = [&](u32 row, float base, float sum, float value_top, bool puts) {
        factors[row] = base;  // the queries' factors and ends are not needed any more
        inverses[row] = sum == 0.0f ? 0.0f : 1.0f / sum;
        row_power[row] = steps(value_top - base);
        if (puts && row < rows && a.lse)
            a.lse[out_row(a, seg, seg.rt * R + row)] = sum == 0.0f ? -INFINITY : (log2f(sum) + base) * kLn2;
    };
    auto put_value = [&](u32 x, float value) {
        const u32 row = x / D;
        if (row >= rows) return;
        const float inverse = inverses[row];  // 0: the row sees nothing
        const float2 f = row_power[row];
        put_out(a, seg, seg.rt * R + row, channel_of(D, x % D), inverse == 0.0f ? 0.0f : value * inverse * f.x * f.y);
    };
    if (threadIdx.x < W * R) {
        const u32 row = threadIdx.x % R;
        float value_top = kNoScore;
#pragma unroll
        for (u32 w = 0; w < W; ++w) value_top = fmaxf(value_top, join_ref[w * R + row]);
        join_factor[threadIdx.x] = steps(join_ref[threadIdx.x] - value_top);
        if (threadIdx.x < R) {
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (u32 w = 0; w < W; ++w) top = fmaxf(top, join_ml[w * R + row].x);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (u32 w = 0; w < W; ++w) sum += join_ml[w * R + row].y * exp2_fast(join_ml[w * R + row].x - base);
            if constexpr (!kWhole) {
                a.part_ml[part * R + row] = make_float2(top, sum);
                a.part_ref[part * R + row] = value_top;
            } else if (team > 1) {
                cta_ml[row] = make_float2(top, sum);
                cta_ref[row] = value_top;
            } else {
                finish_row(row, base, sum, value_top, true);
            }
        }
    }
    __syncthreads();
    for (u32 x = threadIdx.x; x < R * D; x += blockDim.x) {
        const u32 row = x / D, at = x % D;  // `at`: in the joined order
        float value = 0.0f;
#pragma unroll
        for (u32 w = 0; w < W; ++w) {
            const float2 f = join_factor[w * R + row];
            value += join_o[(w * R + row) * (D + 8) + at] * f.x * f.y;
        }
        if constexpr (!kWhole) {
            a.part_o[part * R * D + x] = value;
        } else if (team > 1) {
            cta_o[x] = value;
        } else {
            put_value(x, value);
        }
    }
    float* weights = nullptr;
    if (kWhole && a.weights) {  // one row tile and one list: the weights are this segment's
        weights = a.weights + (static_cast<u64>(seg.seq) * a.c.heads + seg.h) * a.q.width;
        const u32 from = list ? 0 : (seg.tiles + (1u << sub_bits) - 1) >> sub_bits;
        for (u32 j = from + rank * blockDim.x + threadIdx.x; j < a.q.width; j += team * blockDim.x) weights[j] = 0.0f;
    }
    if (team > 1) {
        // join the CTAs, each a run of the values, as the warps were joined
        kv_team_sync(KvTeam{rank, team});
        if (threadIdx.x < team * R) {
            const u32 row = threadIdx.x % R;
            float value_top = kNoScore;
            for (u32 r = 0; r < team; ++r) value_top = fmaxf(value_top, peek(cta_ref + row, r));
            join_factor[threadIdx.x] = steps(peek(cta_ref + row, threadIdx.x / R) - value_top);
            if (threadIdx.x < R) {
                float top = -INFINITY, sum = 0.0f;
                for (u32 r = 0; r < team; ++r) top = fmaxf(top, peek2(cta_ml + row, r).x);
                const float base = top == -INFINITY ? 0.0f : top;
                for (u32 r = 0; r < team; ++r) {
                    const float2 its = peek2(cta_ml + row, r);
                    sum += its.y * exp2_fast(its.x - base);
                }
                finish_row(row, base, sum, value_top, rank == 0);
            }
        }
        __syncthreads();
        const u32 run = R * D / team;
        for (u32 x = rank * run + threadIdx.x; x < (rank + 1) * run; x += blockDim.x) {
            const u32 row = x / D;
            float value = 0.0f;
            for (u32 r = 0; r < team; ++r) {
                const float2 f = join_factor[r * R + row];
                value += peek(cta_o + x, r) * f.x * f.y;
            }
            put_value(x, value);
        }
    }
    __syncthreads();  // before the next segment's copies
    if (weights) {
        // (a CTA of a team without tiles begins where the segment ends, inside a block perhaps)
        const u32 to = first < end ? (end + (1u << sub_bits) - 1) >> sub_bits : 0;
        for (u32 k = (first >> sub_bits) + threadIdx.x; k < to; k += blockDim.x) {
            float w = 0.0f;
            for (u32 t = (k << sub_bits) - first; t < min((k + 1) << sub_bits, end) - first; ++t)
                for (u32 r = 0; r < rows; ++r)
                    w += whole_sums[t * R + r].x * (exp2_fast(whole_sums[t * R + r].y - factors[r]) * inverses[r]);
            const u32 j = list ? static_cast<u32>(list[k]) : k;
            if (j < a.q.width) weights[j] = w;
        }
    }
    if (team > 1) kv_team_sync(KvTeam{rank, team});  // nobody leaves while another may read its sums
}

template <int D, int NT, bool kWhole, u32 W>
__global__ void __launch_bounds__(W * 32, W == kWarps ? per_sm(D, NT) : 1) attention_kernel(const AttentionArgs a)
{
    extern __shared__ __align__(128) u8 smem[];
    using L = Layout<D, NT, W>;
    if constexpr (kWhole) {  // a CTA or a team per segment, which it finishes
        const u32 team = W > kWarps ? a.team : 1u, rank = blockIdx.x % team;
        const Segment seg = segment_of(a, blockIdx.x / team);
        const u32 each = part_of(seg.tiles, team, a.c.block / 16), first = min(rank * each, seg.tiles);
        run_segment<D, NT, true, W>(a, seg, first, min(first + each, seg.tiles), rank, smem);
        return;
    }
    kv_let_next();
    const Place place = place_of(a, reinterpret_cast<u64*>(smem + L::line), reinterpret_cast<Place*>(smem + L::line + 8 * kWarps));
    u64 at = place.at, begin = place.begin;
    const u64 stop = place.stop;
    if (at >= stop) return;
    u32 unit = place.unit;
    u32 tiles = unit_tiles(a, unit);
    while (at < stop) {
        while (tiles == 0 || at >= begin + static_cast<u64>(tiles) * a.per_unit) {
            begin += static_cast<u64>(tiles) * a.per_unit;
            tiles = unit_tiles(a, ++unit);
        }
        const u32 inside = static_cast<u32>((at - begin) / tiles);
        const u64 here = begin + static_cast<u64>(inside) * tiles;
        const Segment seg = segment_of(a, unit * a.per_unit + inside);
        const u32 first = static_cast<u32>(at - here);
        const u32 end = static_cast<u32>(min(stop - here, static_cast<u64>(tiles)));
        if (threadIdx.x == 0) {
            if (first == 0) a.span[seg.index].x = blockIdx.x;
            if (end == tiles) a.span[seg.index].y = blockIdx.x;
        }
        run_segment<D, NT, false, W>(a, seg, first, end, static_cast<u64>(blockIdx.x) + seg.index, smem);
        at = here + end;
    }
}

__device__ __forceinline__ void put_pair(const AttentionArgs& a, u64 at, float x, float y)
{
    if (a.q.type == HBFSIM_KV_BF16)
        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.out) + at) = __floats2bfloat162_rn(x, y);
    else
        *reinterpret_cast<__half2*>(static_cast<__half*>(a.out) + at) = __floats2half2_rn(x, y);
}

// 11 to 16 us by itself (parts and tile sums come out of the L2), of which a
// call shows 2 to 12 us, since its start overlaps the end of the kernel before.
// CTAs (sequence * heads + head, y).  The segments of a (sequence, head) are
// joined by the CTAs y = 0, 1, .. in turn, or, with more CTAs than segments,
// each by `slices` of them; with weights every CTA also sums those of its
// share of the blocks.  All sums run in a fixed order.
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const AttentionArgs a, u32 R, u32 slices)
{
    // of the segment at hand
    __shared__ float row_top[24], row_sum[24], row_inverse[24], row_ref[24];
    __shared__ float4 join[kFinishThreads];
    const u32 i = threadIdx.x, lane = i & 31u, warp = i >> 5;
    kv_wait_before();
    const u32 h = blockIdx.x % a.c.heads, seq = blockIdx.x / a.c.heads;
    const u32 sub_bits = 27 - __clz(a.c.block), D = a.c.dim;
    const u32 each = (a.q.width + gridDim.y - 1) / gridDim.y;
    const u32 from = min(blockIdx.y * each, a.q.width), to_block = min(from + each, a.q.width);
    float* weights = a.tile_sums ? a.weights + (static_cast<u64>(seq) * a.c.heads + h) * a.q.width
                                : nullptr;
    for (u32 n = 0; n < a.lists * a.row_tiles; ++n) {
        u32 slice = n % gridDim.y == blockIdx.y ? 0 : slices;
        if (slices > 1) slice = blockIdx.y - n * slices;  // wraps for CTAs of other segments
        const bool joins = slice < slices;
        if (!joins && !weights) continue;
        const u32 t = n / a.row_tiles, rt = n % a.row_tiles;
        const u32 index = ((seq * a.lists + t) * a.c.heads + h) * a.row_tiles + rt;
        const u32 rows = min(R, a.rows - rt * R);
        const u32 tiles = unit_tiles(a, index / a.per_unit);
        const uint2 span = tiles ? a.span[index] : make_uint2(1, 0);  // its first and last worker
        const u32 parts = span.y + 1 - span.x;
        const u64 first = static_cast<u64>(span.x) + index;
        const float2* ml = a.part_ml + first * R;
        const float* ref = a.part_ref + first * R;
        __syncthreads();
        for (u32 r = warp; r < rows; r += kFinishThreads / 32) {
            float top = -INFINITY, value_top = kNoScore, all = 0.0f;
            for (u32 s = lane; s < parts; s += 32) {
                top = fmaxf(top, ml[s * R + r].x);
                value_top = fmaxf(value_top, ref[s * R + r]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                value_top = fmaxf(value_top, __shfl_xor_sync(0xffffffffu, value_top, o));
            }
            const float base = top == -INFINITY ? 0.0f : top;
            for (u32 s = lane; s < parts; s += 32) all += ml[s * R + r].y * exp2_fast(ml[s * R + r].x - base);
#pragma unroll
            for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            if (lane == 0) {
                row_top[r] = base;
                row_sum[r] = all;
                row_inverse[r] = all == 0.0f ? 0.0f : 1.0f / all;
                row_ref[r] = value_top;
            }
        }
        __syncthreads();
        if (joins) {
            // four channels per thread; groups of threads take the partials in turn
            const u32 all_pieces = rows * D / 4;
            const u32 piece0 = all_pieces * slice / slices;
            const u32 pieces = all_pieces * (slice + 1) / slices - piece0;
            const u32 groups = max(1u, kFinishThreads / pieces);
            const float4* part = reinterpret_cast<const float4*>(a.part_o + first * R * D);
            const u32 group = i / pieces;
            for (u32 at = pieces < kFinishThreads ? i % pieces : i; at < pieces; at += kFinishThreads) {
                const u32 x = piece0 + at, r = x * 4 / D;
                const float base = row_ref[r];
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (group < groups || groups == 1) {
#pragma unroll 8
                    for (u32 s = groups == 1 ? 0 : group; s < parts; s += groups) {
                        const float4 y = part[static_cast<u64>(s) * (R * D / 4) + x];
                        const float by = ref[s * R + r] - base;
                        v.x += at_power(y.x, by);
                        v.y += at_power(y.y, by);
                        v.z += at_power(y.z, by);
                        v.w += at_power(y.w, by);
                    }
                }
                if (groups > 1) {
                    join[i] = v;
                    __syncthreads();  // pieces < kFinishThreads: every thread is here once
                    if (group) break;
                    for (u32 k = 1; k < groups; ++k) {
                        const float4 y = join[k * pieces + at];
                        v.x += y.x;
                        v.y += y.y;
                        v.z += y.z;
                        v.w += y.w;
                    }
                }
                const float by = base - row_top[r];
                auto mean = [&](float x) { return at_power(x * row_inverse[r], by); };
                // two pairs of neighbouring channels, D / 8 apart
                const u32 row = rt * R + r, at_row = x * 4 % D, d = channel_of(D, at_row);
                const u32 tt = a.blocks ? t : row / a.q.group;
                const u32 qh = h * a.q.group + row % a.q.group;
                const u64 to = (static_cast<u64>(seq) * a.q.tokens + tt) * a.q.q_heads + qh;
                put_pair(a, to * D + d, mean(v.x), mean(v.y));
                put_pair(a, to * D + d + D / 8, mean(v.z), mean(v.w));
                if (at_row == 0 && a.lse)
                    a.lse[to] = row_sum[r] == 0.0f ? -INFINITY : (log2f(row_sum[r]) + row_top[r]) * kLn2;
            }
        }
        if (!weights) continue;
        const u32 listed = (tiles + (1u << sub_bits) - 1) >> sub_bits;
        const float2* sums = a.tile_sums + static_cast<u64>(index) * a.tiles * R;
        auto weight_of = [&](u32 k) {
            float w = 0.0f;
            for (u32 tile = k << sub_bits; tile < min((k + 1) << sub_bits, tiles); ++tile) {
                const float4* x = reinterpret_cast<const float4*>(sums + static_cast<u64>(tile) * R);
                for (u32 r = 0; r < rows; r += 2) {
                    const float4 y = x[r / 2];  // two rows' sums and references
                    w += y.x * (exp2_fast(y.y - row_top[r]) * row_inverse[r]);
                    if (r + 1 < rows) w += y.z * (exp2_fast(y.w - row_top[r + 1]) * row_inverse[r + 1]);
                }
            }
            return w;
        };
        if (!a.blocks) {
            for (u32 j = from + i; j < to_block; j += kFinishThreads) {
                const float w = j < listed ? weight_of(j) : 0.0f;
                weights[j] = n ? weights[j] + w : w;  // the same thread's own
            }
        } else {
            const int* list = a.blocks + ((static_cast<u64>(seq) * a.lists + t) * a.c.heads + h) * a.top;
            if (rt == 0 && t == 0)
                for (u32 j = from + i; j < to_block; j += kFinishThreads) weights[j] = 0.0f;
            __syncthreads();
            for (u32 k = i; k < listed; k += kFinishThreads) {
                const u32 j = static_cast<u32>(list[k]);
                if (j >= from && j < to_block) weights[j] += weight_of(k);  // a list names it once
            }
        }
    }
}

Plan plan_of(const KvView& v, const KvQuery& q, const hbfsim_kv_attention_args_v1& g)
{
    return plan_of(PlanCall{q.seqs, q.tokens, v.heads, q.group, v.dim, v.block, q.width, g.top, g.blocks != nullptr,
                            g.weights != nullptr}, static_cast<u32>(kv_sm_count()));
}

int check_args(const hbfsim_kv_attention_args_v1* g)
{
    if (!g || g->struct_size != sizeof(*g) || g->version != HBFSIM_KV_V1_VERSION)
        return HBFSIM_INVALID_ARGUMENT;
    if ((g->blocks == nullptr) != (g->counts == nullptr)) return HBFSIM_INVALID_ARGUMENT;
    if (g->blocks && (g->top == 0 || g->top > kKvMaxWidth)) return HBFSIM_INVALID_ARGUMENT;
    if (!(g->softmax_scale == g->softmax_scale) || g->softmax_scale > 3.0e38f ||
        g->softmax_scale < -3.0e38f)
        return HBFSIM_INVALID_ARGUMENT;
    return HBFSIM_OK;
}

template <int D, int NT, bool kWhole, u32 W>
bool launch_attention(const AttentionArgs& a, cudaStream_t s)
{
    static std::atomic<u64> seen{0};
    using L = Layout<D, NT, W>;
    auto* kernel = attention_kernel<D, NT, kWhole, W>;
    if (!kv_allow_smem(kernel, kWhole ? L::most : L::bytes, seen)) return false;
    const u32 sums = kWhole && a.weights ? part_of(a.tiles, a.team, a.c.block / 16) * 8 * NT * 8 : 0;
    const u32 smem = std::max(L::bytes, L::whole_sums + sums);
    return kv_launch(kernel, dim3(a.workers), W * 32, s, smem, kWhole ? a.team : 1, false, a);
}

template <int D, int NT>
int launch(const AttentionArgs& a, const Plan& p, cudaStream_t s)
{
    if (p.whole) {
        const bool ok = p.warps == kWarps ? launch_attention<D, NT, true, kWarps>(a, s)
                                          : launch_attention<D, NT, true, 2 * kWarps>(a, s);
        return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
    }
    if (!launch_attention<D, NT, false, kWarps>(a, s)) return HBFSIM_CUDA_ERROR;
    // one CTA per segment or more, up to what is resident at once; for the weights no more than
    // have blocks to sum
    const u32 pairs = a.q.seqs * a.c.heads, segments = a.lists * a.row_tiles;
    u32 across = std::max(segments, std::min(segments * 8, 4u * kv_sm_count() / pairs));
    if (a.weights)
        across = std::max(segments, std::min((a.q.width + kFinishThreads - 1) / kFinishThreads,
                                             4u * kv_sm_count() / pairs));
    const u32 slices = std::min(std::max(1u, across / segments), 8u);
    const bool ok = kv_launch(finish_kernel, dim3(pairs, across), kFinishThreads, s, 0, 1, true, a,
                              static_cast<u32>(8 * NT), slices);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" uint64_t hbfsim_kv_attention_workspace_v1(const hbfsim_kv_cache_v1* cache,
                                                     const hbfsim_kv_query_v1* query,
                                                     const hbfsim_kv_attention_args_v1* args)
{
    KvView v{};
    KvQuery q{};
    if (kv_check_cache(cache, v) || kv_check_query(query, v, q) || check_args(args)) return 0;
    if (q.seqs == 0 || q.tokens == 0) return 0;
    return plan_of(v, q, *args).bytes;
}

extern "C" int hbfsim_kv_attention_v1(const hbfsim_kv_cache_v1* cache,
                                      const hbfsim_kv_query_v1* query,
                                      const hbfsim_kv_attention_args_v1* args, void* stream)
{
    AttentionArgs a{};
    if (const int rc = kv_check_cache(cache, a.c)) return rc;
    if (const int rc = kv_check_query(query, a.c, a.q)) return rc;
    if (const int rc = check_args(args)) return rc;
    if (a.q.seqs == 0 || a.q.tokens == 0) return HBFSIM_OK;
    const Plan p = plan_of(a.c, a.q, *args);
    if (p.segments > 0x7fffffffull) return HBFSIM_UNSUPPORTED;
    if (!args->out || (p.bytes && !args->workspace) || args->workspace_bytes < p.bytes ||
        !kv_aligned(args->workspace, 16) || !kv_aligned(args->out, 4) ||
        !kv_aligned(args->lse, 4) || !kv_aligned(args->weights, 4) ||
        !kv_aligned(args->blocks, 4) || !kv_aligned(args->counts, 4))
        return HBFSIM_INVALID_ARGUMENT;
    a.scale2 = args->softmax_scale * kLog2e;
    a.top = args->top;
    a.blocks = args->blocks;
    a.counts = args->counts;
    a.out = args->out;
    a.lse = args->lse;
    a.weights = a.q.width ? args->weights : nullptr;
    a.lists = p.lists;
    a.row_tiles = p.row_tiles;
    a.rows = p.rows;
    a.units = p.units;
    a.per_unit = p.per_unit;
    a.workers = p.workers;
    a.team = p.team;
    a.tiles = p.tiles;
    u8* w = static_cast<u8*>(args->workspace);
    a.part_o = reinterpret_cast<float*>(w + p.part_o);
    a.part_ml = reinterpret_cast<float2*>(w + p.part_ml);
    a.part_ref = reinterpret_cast<float*>(w + p.part_ref);
    a.span = reinterpret_cast<uint2*>(w + p.span);
    a.tile_sums = a.weights && !p.whole ? reinterpret_cast<float2*>(w + p.tile_sums) : nullptr;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (a.c.dim * 8 + p.nt) {
    case 64 * 8 + 1: return launch<64, 1>(a, p, s);
    case 64 * 8 + 2: return launch<64, 2>(a, p, s);
    case 64 * 8 + 3: return launch<64, 3>(a, p, s);
    case 128 * 8 + 1: return launch<128, 1>(a, p, s);
    case 128 * 8 + 2: return launch<128, 2>(a, p, s);
    case 128 * 8 + 3: return launch<128, 3>(a, p, s);
    case 256 * 8 + 1: return launch<256, 1>(a, p, s);
    default: return launch<256, 2>(a, p, s);
    }
}
