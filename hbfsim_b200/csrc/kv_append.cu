// kv_append.cu -- new tokens into the 8-bit paged cache (kv_v1.h).
//
// One warp per (touched block, head, side).  A CTA's warps look at a chunk of
// up to 16 tokens, one per lane, and do the blocks whose first new token is
// among them, each warp for its head and side; few tokens get chunks of one,
// so that every block has a warp of its own at once.  For a block of new
// tokens alone a lane holds its channels of 16 tokens in registers between
// the two passes: the largest magnitude, which gives the scale, then the
// stored values (blocks of more tokens are read again).  Everything is a
// power of two away from the input, so the only rounding is the one to e4m3.
//
// Prompts of 31,668 tokens in all (8 heads of 128 channels) take 42 us: 199 MB
// of input and blocks at 4.8 TB/s, 73 % of a copy's rate.  Nothing is full (56 %
// of the issue slots, 24 warps an SM): a warp loads 16 rows, converts and
// stores them with no other load under way, so latency bounds it.  A step's 64
// tokens take 4.4 us and one token 3.1 us, a launch and one chain of reads
// (start, table, the block's scale, its values).
#include "kv_append.cuh"

namespace hbfb {
namespace {

constexpr u32 kAppendWarps = 4;

template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(kAppendWarps * 32, D == 256 ? 3 : 6) append_kernel(const AppendArgs a)
{
    const u32 pair = blockIdx.y * kAppendWarps + (threadIdx.x >> 5), head = pair >> 1, side = pair & 1u;
    if (head >= a.c.heads) return;
    const Lead mine = lead_of(a, blockIdx.x);
    for (u32 left = __ballot_sync(0xffffffffu, mine.leads); left; left &= left - 1) {
        const int who = __ffs(left) - 1;
        const u32 its_token = blockIdx.x * a.chunk + static_cast<u32>(who);
        const int its_page = __shfl_sync(0xffffffffu, mine.page, who);
        const u32 its_slot = __shfl_sync(0xffffffffu, mine.slot, who);
        const u32 its_count = __shfl_sync(0xffffffffu, mine.count, who);
        append_plain<T, D, kWide>(a, head, side, its_token, its_page, its_slot, its_count);
    }
}

template <typename T>
int launch(const AppendArgs& a, cudaStream_t s)
{
    const dim3 grid((a.tokens + a.chunk - 1) / a.chunk, (a.c.heads * 2 + kAppendWarps - 1) / kAppendWarps);
    auto run = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return kv_launch(a.wide ? append_kernel<T, D, true> : append_kernel<T, D, false>, grid, kAppendWarps * 32, s,
                         0, 1, false, a);
    };
    const bool ok = a.c.dim == 64    ? run(std::integral_constant<int, 64>{})
                    : a.c.dim == 128 ? run(std::integral_constant<int, 128>{})
                                     : run(std::integral_constant<int, 256>{});
    return ok ? HBFSIM_OK : HBFSIM_CUDA_ERROR;
}

}  // namespace
}  // namespace hbfb

using namespace hbfb;

extern "C" int hbfsim_kv_append_v1(const hbfsim_kv_cache_v1* cache,
                                   const hbfsim_kv_append_batch_v1* b, void* stream)
{
    AppendArgs a{};
    if (const int rc = append_check(cache, b, a)) return rc;
    if (b->tokens == 0 || b->width == 0 || a.c.pages == 0) return HBFSIM_OK;  // no block is there
    // One token to a chunk while all chunks' warps are resident at once (16 to an SM), up to 16
    // beyond (8 heads of 128 channels: 64 tokens take 4.4 us with 1, took 26 us with 16, 31,668
    // tokens 145 us with 1 and 42 us with 16).
    a.chunk = 1;
    while (a.chunk < 16 && static_cast<u64>(a.tokens) * a.c.heads * 2 > static_cast<u64>(a.chunk) * 16 * kv_sm_count())
        a.chunk *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return b->type == HBFSIM_KV_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
}
