// kv_verify.cu -- drafted tokens against the target's probabilities (kv_v1.h).
//
// One row of the target (and one of the draft) decides a sequence's next token,
// and which row follows from a few gathered probabilities, so a cluster of up to
// 8 CTAs takes a sequence: every CTA looks up the drafted tokens, reads its slice
// of the row once, and its warps add up whole weights, each over a contiguous
// segment.  The CTAs' sums meet through distributed shared memory; the one whose
// slice holds the border reads the segment that holds it again and finds the
// token.
//
// 64 sequences of 131,072 fp32 values, most of them with a rejected token, take 16.5 us:
// 58 MB in 10 us, and 6 us of latency in front and behind (the gathered probabilities,
// the sums' meeting, the border's segment); in 16 bits 14.5 us for half the bytes.  With
// rows of 1,024 values the call takes 5.0 us.  Rows of 131,071 values, which do not begin
// on 16 bytes, take 18.0 us (fp32) and 16.9 us (bf16).  256 CTAs on 148 SMs leave some with two and some with one; whole numbers
// cost a fifth of the issue slots.  Eight CTAs of 256 threads to a row took 20 us.
#include "kv.h"

#include <type_traits>

namespace hbfb {
namespace {

constexpr u32 kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr u32 kMaxDrafts = 32;
constexpr u32 kMaxVocab = 1u << 22;  // sums stay below 2^62
constexpr u32 kMaxTeam = 8;

struct VerifyArgs {
    const void* target;
    i64 target_seq, target_token;
    const void* draft;
    i64 draft_seq, draft_token;
    const int* tokens;
    const float* accept;
    const float* sample;
    const int* counts;
    const int* lengths;
    int* accepted;
    int* tokens_out;
    int* lengths_out;
    u32 drafts, vocab, segment;  // segment: elements of a warp, a multiple of 256
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// A probability in whole multiples of 2^-40.
__device__ __forceinline__ i64 whole(float p)
{
    return __float2ll_rn(fminf(fmaxf(p, 0.0f), 1.0f) * 1099511627776.0f);  // fmaxf drops NaN; the product is exact
}

// 16 bytes of probabilities, asked for in the order that is written here: the loads of a step are
// all under way before the first is used.
__device__ __forceinline__ uint4 load16(const void* from)
{
    uint4 x;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "l"(from));
    return x;
}

template <typename T>
__device__ __forceinline__ T load_one(const T* from)
{
    if constexpr (sizeof(T) == 4) {
        u32 x;
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(x) : "l"(from));
        return *reinterpret_cast<const T*>(&x);
    } else {
        u16 x;
        asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(x) : "l"(from));
        return *reinterpret_cast<const T*>(&x);
    }
}

struct Sums {
    u64 left, target;  // of the weights, of the target alone
};

template <bool kDraft>
__device__ __forceinline__ void add_to(Sums& s, float p, float q)
{
    const i64 a = whole(p);
    s.target += static_cast<u64>(a);
    if constexpr (kDraft) {
        const i64 d = a - whole(q);
        s.left += static_cast<u64>(d > 0 ? d : 0);
    }
}

// The probabilities of 16 bytes.
template <typename T, bool kDraft>
__device__ __forceinline__ void add_16(Sums& s, const uint4& x, const uint4& y)
{
    const T* p = reinterpret_cast<const T*>(&x);
    const T* q = reinterpret_cast<const T*>(&y);
#pragma unroll
    for (u32 k = 0; k < 16 / sizeof(T); ++k) add_to<kDraft>(s, to_float(p[k]), kDraft ? to_float(q[k]) : 0.0f);
}

// Sums of [from, end) by a warp.
template <typename T, bool kWide, bool kDraft>
__device__ __forceinline__ Sums sum_segment(const T* p, const T* q, u32 from, u32 end)
{
    constexpr u32 N = 16 / sizeof(T), U = kDraft ? 4 : 8;
    const u32 lane = threadIdx.x & 31u;
    Sums s{0, 0};
    if constexpr (kWide) {
        u32 i = from + lane * N;
        for (; i + (U - 1) * 32 * N + N <= end; i += U * 32 * N) {
            uint4 x[U], y[U];
#pragma unroll
            for (u32 u = 0; u < U; ++u) {
                x[u] = load16(p + i + u * 32 * N);
                if constexpr (kDraft) y[u] = load16(q + i + u * 32 * N);
            }
#pragma unroll
            for (u32 u = 0; u < U; ++u) add_16<T, kDraft>(s, x[u], y[u]);
        }
        for (; i + N <= end; i += 32 * N) {
            const uint4 x = load16(p + i), y = kDraft ? load16(q + i) : x;
            add_16<T, kDraft>(s, x, y);
        }
        for (; i < end; ++i)  // one lane's rest
            add_to<kDraft>(s, to_float(p[i]), kDraft ? to_float(q[i]) : 0.0f);
    } else {
        // rows that begin anywhere: one value to a lane and load
        constexpr u32 M = 2 * U;
        u32 i = from + lane;
        for (; i + (M - 1) * 32 < end; i += M * 32) {
            T x[M], y[M];
#pragma unroll
            for (u32 u = 0; u < M; ++u) {
                x[u] = load_one(p + i + u * 32);
                if constexpr (kDraft) y[u] = load_one(q + i + u * 32);
            }
#pragma unroll
            for (u32 u = 0; u < M; ++u) add_to<kDraft>(s, to_float(x[u]), kDraft ? to_float(y[u]) : 0.0f);
        }
        for (; i < end; i += 32) add_to<kDraft>(s, to_float(p[i]), kDraft ? to_float(q[i]) : 0.0f);
    }
    if constexpr (!kDraft) s.left = s.target;
    return s;
}

__device__ __forceinline__ u64 warp_sum(u64 x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// Inclusive prefix sums over a warp.
__device__ __forceinline__ u64 warp_scan(u64 x)
{
    const u32 lane = threadIdx.x & 31u;
#pragma unroll
    for (u32 o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

struct VerifyShared {
    u32 accepted, count;
    int tokens[kMaxDrafts];          // those that were accepted
    int refused;                     // the token that was not accepted, -1 without one
    u64 warp_left[kVerifyWarps], warp_target[kVerifyWarps];
    u64 left, target;                // of the CTA: other CTAs read them
    u64 border;                      // from the segment's beginning on
    u32 segment;                     // the warp's whose segment holds it; kVerifyWarps: none here
    u32 alone;                       // whether the target alone counts
    u64 prefix[kVerifyWarps];
};

template <typename T, bool kWide>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const VerifyArgs a, const u32 size)
{
    __shared__ VerifyShared sm;
    const u32 lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const u32 seq = blockIdx.x / size;
    const KvTeam team{blockIdx.x - seq * size, size};
    const T* target = static_cast<const T*>(a.target) + static_cast<i64>(seq) * a.target_seq;
    const T* draft = static_cast<const T*>(a.draft) + static_cast<i64>(seq) * a.draft_seq;
    float sample = 0.0f;
    int length = 0;
    if (warp == 0) {
        // what does not hang together is asked for at once
        const u64 at = static_cast<u64>(seq) * a.drafts + lane;
        const int given = a.counts ? a.counts[seq] : static_cast<int>(a.drafts);
        int token = lane < a.drafts ? a.tokens[at] : -1;
        const double u = lane < a.drafts ? a.accept[at] : 0.0f;
        sample = a.sample[seq];
        if (a.lengths_out) length = a.lengths[seq];
        const u32 count = static_cast<u32>(min(max(given, 0), static_cast<int>(a.drafts)));
        bool good = false;
        if (static_cast<u32>(token) < a.vocab) {
            const double p = to_float(target[static_cast<i64>(lane) * a.target_token + token]);
            const double q = a.draft ? to_float(draft[static_cast<i64>(lane) * a.draft_token + token]) : 1.0f;
            good = u * q < p;  // 24 bits by 24: exact
        } else {
            token = -1;
        }
        const u32 accepted = __ffs(~__ballot_sync(0xffffffffu, good && lane < count)) - 1u;  // ~0 where all 32 are
        const u32 n = min(accepted, count);
        const int refused = n < count ? __shfl_sync(0xffffffffu, token, static_cast<int>(n)) : -1;
        if (lane == 0) {
            sm.accepted = n;
            sm.count = count;
            sm.refused = refused;
        }
        if (lane < n) sm.tokens[lane] = token;
    }
    __syncthreads();
    const u32 accepted = sm.accepted;
    const bool rejected = accepted < sm.count;
    int* out = a.tokens_out + static_cast<u64>(seq) * (a.drafts + 1);
    const T* p = target + static_cast<i64>(accepted) * a.target_token;
    const T* q = rejected && a.draft ? draft + static_cast<i64>(accepted) * a.draft_token : nullptr;
    const u32 refused = rejected && !a.draft ? static_cast<u32>(sm.refused) : ~0u;
    auto bounds = [&](u32 segment, u32& from, u32& end) {
        const u64 at = static_cast<u64>(team.rank * kVerifyWarps + segment) * a.segment;
        from = static_cast<u32>(min(at, static_cast<u64>(a.vocab)));
        end = static_cast<u32>(min(at + a.segment, static_cast<u64>(a.vocab)));
    };
    u32 from, end;
    bounds(warp, from, end);
    Sums s = q ? sum_segment<T, kWide, true>(p, q, from, end) : sum_segment<T, kWide, false>(p, q, from, end);
    s.left = warp_sum(s.left);
    s.target = warp_sum(s.target);
    if (lane == 0) {
        if (refused >= from && refused < end) s.left -= static_cast<u64>(whole(to_float(p[refused])));
        sm.warp_left[warp] = s.left;
        sm.warp_target[warp] = s.target;
    }
    __syncthreads();
    if (warp == 0) {
        const u64 l = warp_sum(lane < kVerifyWarps ? sm.warp_left[lane] : 0);
        const u64 t = warp_sum(lane < kVerifyWarps ? sm.warp_target[lane] : 0);
        if (lane == 0) {
            sm.left = l;
            sm.target = t;
        }
    }
    auto find = [&]() {
        if (sm.segment == kVerifyWarps) return;
        // the segment again, a run of neighbours to a thread
        bounds(sm.segment, from, end);
        const u32 each = (end - from + kVerifyThreads - 1) / kVerifyThreads;
        const u32 first = min(from + threadIdx.x * each, end), last = min(first + each, end);
        const bool alone = sm.alone != 0;
        auto weight_at = [&](u32 i) {
            const i64 x = whole(to_float(p[i]));
            if (alone) return static_cast<u64>(x);
            if (i == refused) return u64{0};
            const i64 d = q ? x - whole(to_float(q[i])) : x;
            return static_cast<u64>(d > 0 ? d : 0);
        };
        u64 mine = 0;
        for (u32 i = first; i < last; ++i) mine += weight_at(i);
        const u64 upto = warp_scan(mine);
        if (lane == 31) sm.prefix[warp] = upto;
        __syncthreads();
        u64 before = upto - mine;
        for (u32 w = 0; w < warp; ++w) before += sm.prefix[w];
        const u64 border = sm.border;
        if (border < before || border >= before + mine) return;
        for (u32 i = first; i < last; ++i) {
            before += weight_at(i);
            if (border < before) {
                out[accepted] = static_cast<int>(i);
                return;
            }
        }
    };
    kv_team_sync(team);
    if (warp == 0) {
        u64 l = lane == 0 ? sm.left : 0, t = lane == 0 ? sm.target : 0;
        if (size > 1) {
            l = lane < size ? kv_peek(&sm.left, lane) : 0;
            t = lane < size ? kv_peek(&sm.target, lane) : 0;
        }
        if (size > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        const bool alone = warp_sum(l) == 0;
        const u64 mine = alone ? t : l, sum = warp_sum(mine), upto = warp_scan(mine);
        const u64 before = __shfl_sync(0xffffffffu, upto - mine, static_cast<int>(size > 1 ? team.rank : 0));
        // floor(u * sum / 2^24), sum < 2^62
        const u32 u = static_cast<u32>(fminf(fmaxf(sample, 0.0f) * 16777216.0f, 16777215.0f));
        const u64 border = (u * (sum >> 32) << 8) + (u * (sum & 0xffffffffu) >> 24);
        // the segment of this CTA that holds it
        const u64 weight = lane < kVerifyWarps ? (alone ? sm.warp_target[lane] : sm.warp_left[lane]) : 0;
        const u64 inclusive = before + warp_scan(weight);
        const bool here = sum > 0 && border < inclusive && border >= inclusive - weight;
        const u32 who = __ballot_sync(0xffffffffu, here);
        if (here) sm.border = border - (inclusive - weight);
        if (lane == 0) {
            sm.segment = who ? static_cast<u32>(__ffs(who) - 1) : kVerifyWarps;
            sm.alone = alone;
        }
        if (team.rank == 0) {
            for (u32 i = lane; i <= a.drafts; i += 32)
                if (i != accepted || sum == 0) out[i] = i < accepted ? sm.tokens[i] : -1;
            if (lane == 0) {
                a.accepted[seq] = static_cast<int>(accepted);
                if (a.lengths_out) a.lengths_out[seq] = length - static_cast<int>(sm.count - accepted);
            }
        }
    } else if (size > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    }
    __syncthreads();
    find();
    // nobody leaves while another may read its sums
    if (size > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T>
bool launch(VerifyArgs& a, u32 seqs, cudaStream_t s)
{
    constexpr u32 N = 16 / sizeof(T);
    auto wide = [&](const void* p, i64 seq, i64 token) {
        return kv_aligned(p, 16) && seq % N == 0 && token % N == 0;
    };
    const bool all = wide(a.target, a.target_seq, a.target_token) &&
                     (!a.draft || wide(a.draft, a.draft_seq, a.draft_token));
    // CTAs to a sequence: a power of two, as long as all are resident at once (two to an SM, less what
    // clusters leave unused) and each has 4096 values or more.
    u32 team = 1;
    while (team < kMaxTeam && static_cast<u64>(seqs) * team * 2 <= static_cast<u64>(kv_sm_count()) * 7 / 4 &&
           a.vocab / (team * 2) >= 4096)
        team *= 2;
    a.segment = (a.vocab + team * kVerifyWarps * 256 - 1) / (team * kVerifyWarps * 256) * 256;
    return kv_launch(all ? verify_kernel<T, true> : verify_kernel<T, false>, dim3(seqs * team), kVerifyThreads, s, 0,
                     team, false, a, team);
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" int hbfsim_kv_verify_v1(const hbfsim_kv_verify_batch_v1* b, void* stream)
{
    if (!b || b->struct_size != sizeof(*b) || b->version != HBFSIM_KV_V1_VERSION) return HBFSIM_INVALID_ARGUMENT;
    if (b->type > HBFSIM_KV_P_F32 || b->drafts > kMaxDrafts) return HBFSIM_UNSUPPORTED;
    if (b->seqs > kKvMaxSeqs || b->vocab == 0 || b->vocab > kMaxVocab) return HBFSIM_INVALID_ARGUMENT;
    if (b->seqs == 0) return HBFSIM_OK;
    if (!b->target || !b->sample || !b->accepted || !b->tokens_out || (b->drafts && (!b->tokens || !b->accept)) ||
        (b->lengths_out && !b->lengths))
        return HBFSIM_INVALID_ARGUMENT;
    const u32 size = b->type == HBFSIM_KV_P_F32 ? 4 : 2;
    if (!kv_aligned(b->target, size) || !kv_aligned(b->draft, size) || !kv_aligned(b->tokens, 4) ||
        !kv_aligned(b->accept, 4) || !kv_aligned(b->sample, 4) || !kv_aligned(b->counts, 4) ||
        !kv_aligned(b->lengths, 4) || !kv_aligned(b->accepted, 4) || !kv_aligned(b->tokens_out, 4) ||
        !kv_aligned(b->lengths_out, 4))
        return HBFSIM_INVALID_ARGUMENT;
    // a sequence's own count and length are read before its outputs are written
    const u64 seqs = b->seqs, per_seq = seqs * 4, per_draft = per_seq * b->drafts;
    const KvExtent out[] = {{b->accepted, per_seq}, {b->tokens_out, per_draft + per_seq},
                            {b->lengths_out, b->lengths_out ? per_seq : 0}};
    const KvExtent in[] = {{b->counts, b->counts ? per_seq : 0},
                           {b->lengths, b->lengths_out ? per_seq : 0},
                           {b->tokens, per_draft},
                           {b->accept, per_draft},
                           {b->sample, per_seq},
                           {b->target, seqs, b->target_stride_seq, b->drafts + 1ull, b->target_stride_token, b->vocab, size},
                           {b->draft, b->draft ? seqs : 0, b->draft_stride_seq, b->drafts, b->draft_stride_token, b->vocab,
                            size}};
    if (kv_would_race(out, in, {0, -1, 1})) return HBFSIM_INVALID_ARGUMENT;
    VerifyArgs a{b->target, b->target_stride_seq, b->target_stride_token, b->draft, b->draft_stride_seq,
                 b->draft_stride_token, b->tokens, b->accept, b->sample, b->counts, b->lengths, b->accepted,
                 b->tokens_out, b->lengths_out, b->drafts, b->vocab, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool ok = b->type == HBFSIM_KV_P_F32    ? launch<float>(a, b->seqs, s)
                    : b->type == HBFSIM_KV_P_BF16 ? launch<__nv_bfloat16>(a, b->seqs, s)
                                                  : launch<__half>(a, b->seqs, s);
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}
