"""The operators over the 8-bit paged key/value cache (include/hbfsim/kv_v1.h)
against their definitions in 64 bits (oracle/kv_oracle.py).

What is stored, listed or evicted has to be equal: every rounding there is
part of the definition.  The bounds on the attention's floating outputs:

  scores   products of f16 values are exact; at most 256 of them are added in
           fp32, each addition off by at most 2^-23 of the largest partial
           sum, so a score is off by d = 2^-15 * reach at the very most
           (256 * 2^-23, reach: the row's largest sum of |products|); typical
           errors are a hundred times smaller, and d = 2^-19 * reach is asked
  exp, log 2^-21 relative
  out      2^-11 from rounding the probabilities to f16 and 2 d + 2^-20 from
           the above, of mass (the softmax mean of |values|); 2^-25 of the
           largest value a token that f16 cannot hold normally; and the
           output type's half unit (2^-8 bf16, 2^-11 f16)
  lse      d + 2^-20 (1 + |lse|);   weights  2 d + 2^-19 relative
"""
import itertools

import numpy as np
import pytest

import kv_oracle as ko

pytestmark = pytest.mark.gpu


def torch_():
    import torch
    return torch


def type_of(name):
    torch = torch_()
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def random_cache(rng, pages, heads, block, dim, nan_share=0.0):
    """Values with strong channels and block sizes that differ; bounds of all tokens."""
    x = rng.standard_normal((pages, heads, 2, block, dim))
    x *= np.exp(0.5 * rng.standard_normal((1, heads, 2, 1, dim)))
    x *= np.exp(rng.standard_normal((pages, heads, 2, 1, 1)))
    scale = np.empty((pages, heads, 2))
    for p, h, s in itertools.product(range(pages), range(heads), range(2)):
        scale[p, h, s] = 2.0 ** ko.scale_exponent(np.abs(x[p, h, s]).max())
    data = ko.encode(x / scale[..., None, None])
    key = ko.E4M3[data[:, :, 0]]
    bounds = np.stack([np.floor(key.min(2) / 4), np.ceil(key.max(2) / 4)], 2).astype(np.int8)
    return {"data": data, "scale": scale, "bounds": bounds}


def to_gpu(cache):
    torch = torch_()
    from hbfsim_b200 import KvCache
    return KvCache(torch.from_numpy(cache["data"]).cuda().view(torch.float8_e4m3fn),
                   torch.from_numpy(cache["scale"].astype(np.float32)).cuda(),
                   torch.from_numpy(cache["bounds"]).cuda())


def from_gpu(c):
    torch = torch_()
    return {"data": c.data.view(torch.uint8).cpu().numpy(),
            "scale": c.scale.double().cpu().numpy(), "bounds": c.bounds.cpu().numpy()}


def make_table(rng, lengths, block, pages, extra=0):
    """Blocks of the sequences at random pages, -1 behind; entries past a length are
    poison where the table is wider."""
    have = [-(-max(0, n) // block) for n in lengths]
    width = max(1, max(have, default=1)) + extra
    order = rng.permutation(pages)
    table = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for b, n in enumerate(have):
        table[b, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table


def int32(x):
    return torch_().from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def same_values(got, want, what):
    a, b = ko.E4M3[got], ko.E4M3[want]
    assert np.array_equal(a, b, equal_nan=True), what


def same_cache(c, want):
    got = from_gpu(c)
    same_values(got["data"], want["data"], "data")
    assert np.array_equal(got["scale"], want["scale"]), "scale"
    assert np.array_equal(got["bounds"], want["bounds"]), "bounds"


# ---------------------------------------------------------------------------
# append

APPENDS = [  # dim, block, heads, type, (start, new) per sequence
    (128, 16, 2, "bf16", [(0, 1)]),
    (64, 16, 1, "f16", [(15, 1), (16, 1), (17, 1), (0, 0)]),
    (128, 16, 8, "bf16", [(5, 40), (0, 16), (31, 1), (16, 17), (7, 0), (100, 3)]),
    (256, 32, 3, "f16", [(30, 5), (0, 33), (64, 64)]),
    (64, 64, 2, "bf16", [(63, 2), (1, 200)]),
]


@pytest.mark.parametrize("dim,block,heads,kind,what", APPENDS)
def test_append(dim, block, heads, kind, what):
    torch = torch_()
    from hbfsim_b200 import kv_append
    rng = np.random.default_rng(dim + block + heads)
    start = np.array([s for s, _ in what], np.int32)
    count = np.array([n for _, n in what])
    offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    lengths = start + count
    pages = int(sum(-(-n // block) for n in lengths)) + 2
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, lengths, block, pages, extra=1)
    total = int(offsets[-1])
    # keys and values as slices of one projection, sizes from tiny to huge
    x = rng.standard_normal((total, 3 * heads, dim)) * 10.0 ** rng.uniform(-3, 3, (total, 3 * heads, 1))
    qkv = torch.from_numpy(x).to(type_of(kind)).cuda()
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    gpu = to_gpu(cache)
    for _ in range(2):  # the same tokens again leave everything as it is
        kv_append(gpu, k, v, int32(table), int32(start), offsets=int32(offsets))
        ko.append(cache, k.double().cpu().numpy(), v.double().cpu().numpy(), table, start, offsets)
        same_cache(gpu, cache)


def test_append_uniform_and_odd_strides():
    """[seqs, n, heads, dim] without offsets; a view whose rows start at odd elements."""
    torch = torch_()
    from hbfsim_b200 import kv_append
    rng = np.random.default_rng(5)
    heads, dim, block, seqs, n = 2, 64, 16, 3, 4
    start = np.array([14, 0, 29], np.int32)
    cache = random_cache(rng, 10, heads, block, dim)
    table = make_table(rng, start + n, block, 10)
    wide = torch.from_numpy(rng.standard_normal((seqs * n, heads, dim + 3))).to(torch.bfloat16).cuda()
    k = wide[:, :, 1:dim + 1].unflatten(0, (seqs, n))
    v = wide[:, :, 3:].unflatten(0, (seqs, n))
    gpu = to_gpu(cache)
    kv_append(gpu, k, v, int32(table), int32(start))
    flat = lambda t: t.double().cpu().numpy().reshape(seqs * n, heads, dim)
    ko.append(cache, flat(k), flat(v), table, start, np.arange(seqs + 1) * n)
    same_cache(gpu, cache)


def test_append_special_values():
    """Zeros, infinities, NaN, subnormals and the largest bfloat16; a scale that grows over
    earlier tokens; a rollback (start inside what was written); blocks that are not there."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_append
    heads, dim, block = 1, 64, 16
    gpu = KvCache.empty(4, heads, dim, block)
    cache = from_gpu(gpu)
    table = np.array([[2, 0, -1, 99], [1, 3, -5, 4]], np.int32)  # 99, 4: past the pool
    inf, nan = float("inf"), float("nan")
    big = 3.3895e38
    steps = [
        (np.array([0, 0]), [0.0, 1.0]), (np.array([1, 1]), [inf, 2.0]),
        (np.array([2, 2]), [nan, 1e-30]), (np.array([3, 3]), [1e-40, 3e4]),
        (np.array([4, 4]), [big, -big]), (np.array([2, 1]), [1.0, 448.0]),
        (np.array([15, 16]), [7.0, nan]), (np.array([31, 31]), [5.0, inf]),
        (np.array([32, 40]), [1.0, 1.0]), (np.array([63, 64]), [1.0, 1.0]),
    ]
    for start, value in steps:
        x = torch.tensor(value, dtype=torch.float32).view(2, 1, 1, 1).expand(2, 1, heads, dim).clone()
        x[:, :, :, 1::2] *= 0.37
        x[:, :, :, 2::5] *= -1
        x = x.to(torch.bfloat16).cuda()
        kv_append(gpu, x, x, int32(table), int32(start))
        flat = x.double().cpu().numpy().reshape(2, heads, dim)
        ko.append(cache, flat, flat, table, start, np.array([0, 1, 2]))
        same_cache(gpu, cache)


# ---------------------------------------------------------------------------
# attention


def attend_and_check(cache, q, table, lengths, lists=None, scale=None, gpu=None, weights=True,
                     stream=None):
    """q: CUDA tensor; lists: per (b, t, h) Python lists (a -7 stands for junk)."""
    torch = torch_()
    from hbfsim_b200 import kv_attention
    gpu = gpu or to_gpu(cache)
    B, n, Hq, D = q.shape
    blocks = counts = None
    if lists is not None:
        heads = gpu.kv_heads
        top = max(1, max((len(x) for b in lists for t in b for x in t), default=1)) + 1
        blocks = np.full((B, n, heads, top), 1 << 30, np.int32)  # junk behind the counts
        counts = np.zeros((B, n, heads), np.int32)
        for b, t, h in itertools.product(range(B), range(n), range(heads)):
            counts[b, t, h] = len(lists[b][t][h])
            blocks[b, t, h, :counts[b, t, h]] = lists[b][t][h]
        blocks, counts = int32(blocks), int32(counts)
    got = kv_attention(gpu, q, table if hasattr(table, "cuda") else int32(table), int32(lengths),
                       scale=scale, blocks=blocks, counts=counts, weights=weights, stream=stream)
    torch.cuda.synchronize()
    want = ko.attention(cache, q.double().cpu().numpy(),
                        table.cpu().numpy() if hasattr(table, "cuda") else table, lengths,
                        D ** -0.5 if scale is None else scale, lists)
    out, lse, mass_w, mass, reach, vmax = want
    d = 2.0 ** -19 * reach
    unit = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    tol = (unit * np.abs(out) + (2.0 ** -11 + 2 * d + 2.0 ** -20)[..., None] * mass * (1 + unit)
           + 2.0 ** -25 * (1 + vmax[..., None] * table.shape[1] * gpu.block_tokens))
    go = got.out.double().cpu().numpy()
    most = torch.finfo(q.dtype).max
    past = np.abs(out) + tol > most  # may round to the type's infinity
    assert (np.isfinite(go) | past).all() and (np.sign(go) == np.sign(out))[past].all()
    off = np.abs(np.clip(go, -most, most) - np.clip(out, -most, most))
    assert (off <= tol).all(), f"out: {np.nanmax(off / tol)} times the bound"
    gl = got.lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(gl), np.isneginf(lse)), "rows that see nothing"
    fine = ~np.isneginf(lse)
    off = np.abs(gl[fine] - lse[fine])
    tol = d[fine] + 2.0 ** -20 * (1 + np.abs(lse[fine]))
    assert (off <= tol).all(), f"lse: {np.max(off / tol)} times the bound"
    if weights:
        gw = got.weights.double().cpu().numpy()
        off, tol = np.abs(gw - mass_w), mass_w * (2 * d.max() + 2.0 ** -19) + 1e-30
        assert (off <= tol).all(), f"weights: {np.max(off / tol)} times the bound"
    else:
        assert got.weights is None
    return got


ATTENDS = [  # dim, block, heads, group, tokens, type, lengths
    (64, 16, 1, 8, 1, "f16", [301]),
    (128, 16, 2, 4, 1, "bf16", [1, 15, 16, 17, 0, 32, 33, 100]),
    (128, 16, 8, 4, 1, "bf16", [1999, 3]),
    (256, 16, 2, 2, 1, "f16", [130, 7]),
    (64, 32, 3, 7, 3, "bf16", [2, 3, 31, 64, 65, 0, 200]),
    (128, 64, 2, 1, 5, "f16", [4, 5, 63, 66, 129]),
    (128, 16, 1, 8, 5, "bf16", [1, 4, 16, 21, 500]),
    (256, 64, 1, 16, 2, "bf16", [1, 90]),
    (64, 16, 2, 64, 1, "f16", [50, 16]),
    (128, 32, 1, 12, 16, "f16", [10, 16, 40]),
    (64, 16, 1, 1, 1, "bf16", [5000]),
    (64, 16, 2, 8, 3, "f16", [700, 23]),
    (128, 16, 1, 8, 4, "bf16", [333]),
    (256, 32, 1, 4, 6, "f16", [450, 6]),
]


@pytest.mark.parametrize("extra", [3, 40])
@pytest.mark.parametrize("dim,block,heads,group,tokens,kind,lengths", ATTENDS)
def test_attention(dim, block, heads, group, tokens, kind, lengths, extra):
    """extra: blocks that the table has room for beyond the longest sequence (short rows are
    finished by one kernel, wider ones are shared out and joined)."""
    torch = torch_()
    rng = np.random.default_rng(dim + block + heads + group + tokens)
    pages = int(sum(-(-n // block) for n in lengths)) + 2
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, lengths, block, pages, extra=extra)
    # what no token uses is NaN
    for b, n in enumerate(lengths):
        if n % block:
            cache["data"][table[b, n // block], :, :, n % block:] = 0x7f
    cache["data"][sorted(set(range(pages)) - set(table.ravel().tolist()))] = 0x7f
    x = 1.5 * rng.standard_normal((len(lengths), tokens, (group + 2) * heads, dim))
    q = torch.from_numpy(x).to(type_of(kind)).cuda()[:, :, :group * heads]
    got = attend_and_check(cache, q, table, lengths)
    again = attend_and_check(cache, q, table, lengths)
    for a, b in zip(got, again):  # the same bits again
        assert torch.equal(a, b)
    # lists: all blocks in another order give the same; then some of them, and none
    have = [-(-n // block) for n in lengths]
    for share in (1.0, 0.4, 0.0):
        lists = [[[[int(j) for j in rng.permutation(have[b]) if rng.random() < share]
                   for _ in range(heads)] for _ in range(tokens)] for b in range(len(lengths))]
        attend_and_check(cache, q, table, lengths, lists)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_splits_a_long_sequence(kind):
    """Few rows and many blocks: the work is split along the sequence; a row whose largest
    scores all lie in one share; values of very different block scales (some outputs are past
    f16's range)."""
    torch = torch_()
    rng = np.random.default_rng(11)
    dim, block, heads, n = 64, 16, 1, 20011
    pages = -(-n // block)
    cache = random_cache(rng, pages, heads, block, dim)
    cache["scale"][:, :, 1] *= 2.0 ** rng.integers(-20, 21, (pages, heads))
    table = make_table(rng, [n], block, pages)
    q = torch.from_numpy(3 * rng.standard_normal((1, 1, 4, dim))).to(type_of(kind)).cuda()
    attend_and_check(cache, q, table, [n])


def test_attention_holes_and_lists_of_absent_blocks():
    torch = torch_()
    rng = np.random.default_rng(12)
    dim, block, heads, group = 128, 16, 2, 4
    lengths = [200, 64, 33]
    pages = 30
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, lengths, block, pages, extra=2)
    table[0, [0, 5]] = -1
    table[0, 3] = pages           # past the pool
    table[1, :] = -1              # nothing there at all
    q = torch.from_numpy(rng.standard_normal((3, 2, heads * group, dim))).to(torch.bfloat16).cuda()
    got = attend_and_check(cache, q, table, lengths)
    assert not got.out[1].any() and torch.isneginf(got.lse[1]).all() and not got.weights[1].any()
    lists = [[[[0, 1, -7, 12, 13, 1 << 29]] * heads] * 2, [[[0]] * heads] * 2,
             [[[2, 1]] * heads, [[]] * heads]]
    attend_and_check(cache, q, table, lengths, lists)


@pytest.mark.parametrize("q_size,key_exp,value_exp", [(1e30, -90, 100), (1e-30, 60, -100), (50, 0, 0)])
def test_attention_extreme_sizes(q_size, key_exp, value_exp):
    """Queries beyond f16's range, block scales near their limits, sharp softmaxes."""
    torch = torch_()
    rng = np.random.default_rng(13)
    dim, block, heads = 64, 16, 2
    cache = random_cache(rng, 20, heads, block, dim)
    cache["scale"] = cache["scale"] * 0 + 2.0 ** rng.integers(-2, 3, cache["scale"].shape)
    cache["scale"][:, :, 0] *= 2.0 ** key_exp
    cache["scale"][:, :, 1] *= 2.0 ** value_exp
    table = make_table(rng, [300], block, 20)
    q = torch.from_numpy(q_size * rng.standard_normal((1, 1, 6, dim))).to(torch.bfloat16).cuda()
    scale = 1.0 / (q_size * 2.0 ** key_exp * 448 * 4)
    attend_and_check(cache, q, table, [300], scale=scale)
    attend_and_check(cache, q, table, [300], scale=-scale)


@pytest.mark.parametrize("dim,group,tokens,extra", [(64, 2, 6, 0), (128, 8, 4, 40), (256, 3, 5, 0),
                                                    (128, 4, 2, 0)])
def test_attention_nan_stays_in_the_rows_that_see_it(dim, group, tokens, extra):
    """A key and a value that are NaN at the last positions: earlier query tokens must not
    meet them, later ones do."""
    torch = torch_()
    from hbfsim_b200 import kv_attention
    rng = np.random.default_rng(14)
    block, heads, n = 16, 1, 40
    cache = random_cache(rng, 3, heads, block, dim)
    table = make_table(rng, [n], block, 3, extra=extra)
    q = torch.from_numpy(rng.standard_normal((1, tokens, group, dim))).to(torch.float16).cuda()
    clean = attend_and_check(cache, q, table, [n], weights=False)
    for side in (0, 1):
        for position in (n - 1, n - 3):
            bad = {k: v.copy() for k, v in cache.items()}
            bad["data"][table[0, position // block], 0, side, position % block] = 0x7f
            got = kv_attention(to_gpu(bad), q, int32(table), int32([n]))
            sees = torch.arange(n - tokens, n) >= position
            assert torch.isnan(got.out[0, sees]).all()
            assert torch.equal(got.out[0, ~sees], clean.out[0, ~sees])
            assert torch.isfinite(got.lse[0, ~sees]).all()


def test_attention_views_stream_and_graph():
    """A table that is a slice of a wider one, queries with odd strides, another stream, and a
    captured graph replayed on new contents."""
    torch = torch_()
    from hbfsim_b200 import kv_attention, kv_select
    rng = np.random.default_rng(15)
    dim, block, heads, group = 128, 16, 2, 4
    lengths = [77, 160]
    cache = random_cache(rng, 20, heads, block, dim)
    table = make_table(rng, lengths, block, 20)
    wide = int32(np.concatenate([np.full((2, 3), 5), table, np.full((2, 2), 7)], 1))
    view = wide[:, 3:3 + table.shape[1]]
    x = torch.from_numpy(rng.standard_normal((2, 2, heads * group, dim + 1))).to(torch.bfloat16).cuda()
    q = x[..., 1:]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    attend_and_check(cache, q, view, lengths, stream=stream)
    gpu = to_gpu(cache)
    lens = int32(lengths)
    q = q.contiguous()
    kv_attention(gpu, q, view, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pick = kv_select(gpu, q, view, lens, top=4)
        got = kv_attention(gpu, q, view, lens, blocks=pick.blocks, counts=pick.counts, weights=True)
    for seed in (1, 2):
        q.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal(tuple(q.shape))))
        graph.replay()
        torch.cuda.synchronize()
        want = kv_attention(gpu, q, view, lens, blocks=pick.blocks, counts=pick.counts, weights=True)
        lists = ko.select(cache, q.double().cpu().numpy(), table, lengths, 4, 1, 1)
        assert_lists(pick, lists)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_pool_past_32_bit_offsets():
    """Pages whose bytes lie beyond 2^32: append, select and attend there."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_append, kv_attention, kv_select
    heads, dim, block = 1, 128, 16
    pages = (1 << 32) // 4096 + 1000
    rng = np.random.default_rng(16)
    gpu = KvCache.empty(pages, heads, dim, block)
    n = 100
    own = pages - 1 - np.arange(-(-n // block))
    table = own[None].astype(np.int32)
    x = torch.from_numpy(rng.standard_normal((1, n, heads, dim))).to(torch.bfloat16).cuda()
    kv_append(gpu, x, x * 2, int32(table), int32([0]))
    small = {"data": np.zeros((own.size, heads, 2, block, dim), np.uint8),
             "scale": np.ones((own.size, heads, 2)),
             "bounds": np.zeros((own.size, heads, 2, dim), np.int8)}
    near = np.arange(own.size)[None].astype(np.int32)
    flat = x.double().cpu().numpy()[0]
    ko.append(small, flat, 2 * flat, near, np.array([0]), np.array([0, n]))
    at = torch.from_numpy(own).cuda()
    same_values(gpu.data.view(torch.uint8)[at].cpu().numpy(), small["data"], "data")
    q = torch.from_numpy(rng.standard_normal((1, 1, 4, dim))).to(torch.bfloat16).cuda()
    pick = kv_select(gpu, q, int32(table), int32([n]), top=3)
    assert_lists(pick, ko.select(small, q.double().cpu().numpy(), near, [n], 3, 1, 1))
    far = kv_attention(gpu, q, int32(table), int32([n]), weights=True)
    want = attend_and_check(small, q, near, [n])
    for a, b in zip(far, want):
        assert torch.equal(a, b)


def test_nothing_there():
    """A pool without pages, a table without columns, no sequences, no query tokens: outputs are
    what they are for a query that sees nothing."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_append, kv_attention, kv_evict, kv_select
    q = torch.ones((2, 1, 4, 64), dtype=torch.float16, device="cuda")
    k = torch.ones((2, 1, 2, 64), dtype=torch.float16, device="cuda")
    for pages, width in ((0, 3), (4, 0), (0, 0), (0, 3000)):
        gpu = KvCache.empty(pages, 2, 64)
        table = torch.zeros((2, width), dtype=torch.int32, device="cuda")
        lengths = int32([20, 40])
        kv_append(gpu, k, k, table, lengths)
        got = kv_attention(gpu, q, table, lengths, weights=True)
        assert not got.out.any() and torch.isneginf(got.lse).all() and not got.weights.any()
        pick = kv_select(gpu, q, table, lengths, top=3)
        assert (pick.blocks == -1).all() and not pick.counts.any()
        got = kv_attention(gpu, q, table, lengths, blocks=pick.blocks, counts=pick.counts, weights=True)
        assert not got.out.any() and torch.isneginf(got.lse).all() and not got.weights.any()
    gpu = KvCache.empty(4, 2, 64)
    none = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    assert kv_attention(gpu, q[:0], none, int32([]), weights=True).weights.shape == (0, 2, 3)
    assert kv_select(gpu, q[:0], none, int32([]), top=2).blocks.shape == (0, 1, 2, 2)
    kv_append(gpu, k[:0], k[:0], none, int32([]))
    table = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    got = kv_attention(gpu, q[:, :0], table, int32([3, 3]), weights=True)
    assert got.out.shape == (2, 0, 4, 64) and not got.weights.any()
    rest = kv_evict(torch.zeros((2, 0), dtype=torch.int64, device="cuda"),
                    torch.zeros((2, 1, 0), device="cuda"), table[:, :0], int32([5, 0]), keep=2)
    assert rest.lengths.tolist() == [0, 0] and rest.freed_counts.tolist() == [0, 0]


def test_many_sequences():
    """More (sequence, head) pairs than a grid's second axis holds."""
    torch = torch_()
    from hbfsim_b200 import kv_attention, kv_evict, kv_select
    rng = np.random.default_rng(17)
    seqs, heads, dim, block = 40000, 2, 64, 16
    small = random_cache(rng, 8, heads, block, dim)
    table = rng.integers(0, 8, (seqs, 2)).astype(np.int32)
    lengths = rng.integers(0, 33, seqs)
    q = torch.from_numpy(rng.standard_normal((64, 1, 2 * heads, dim))).to(torch.bfloat16).cuda()
    q = q.repeat(seqs // 64, 1, 1, 1)
    gpu = to_gpu(small)
    wide = np.concatenate([table, np.full((seqs, 40), -1, np.int32)], 1)
    probe = rng.integers(0, seqs, 50)
    want = ko.attention(small, q[probe].double().cpu().numpy(), table[probe], lengths[probe], dim ** -0.5)
    for t in (table, wide):
        got = kv_attention(gpu, q, int32(t), int32(lengths), weights=True)
        assert np.abs(got.out[probe].double().cpu().numpy() - want[0]).max() <= \
            (2.0 ** -8 * np.abs(want[0]) + 2.0 ** -10 * want[3] + 2.0 ** -20).max()
        assert np.abs(got.weights[probe][..., :2].double().cpu().numpy() - want[2]).max() <= 2.0 ** -17
        pick = kv_select(gpu, q, int32(t), int32(lengths), top=2)
        assert np.array_equal(pick.counts.cpu().numpy()[:, 0, 0], -(-lengths // block))
    rest = kv_evict(torch.zeros((seqs, 2), dtype=torch.int64, device="cuda"),
                    torch.rand((seqs, heads, 2), device="cuda"), int32(table), int32(lengths), keep=2)
    assert not rest.freed_counts.any()


@pytest.mark.parametrize("dim, block, heads, group, kind", [
    (128, 16, 4, 4, "bf16"), (64, 32, 5, 8, "f16"), (256, 16, 4, 1, "bf16"), (128, 16, 8, 2, "f16"),
    (64, 64, 9, 5, "bf16"), (128, 32, 5, 16, "bf16"), (256, 32, 4, 13, "f16"), (64, 16, 4, 24, "f16")])
def test_attention_many_short_rows(dim, block, heads, group, kind):
    """Enough (sequence, head) pairs for each to be finished by one thread block up to 70 tiles of
    16 tokens; the same rows shared out and joined, in a wider table; lists of them."""
    torch = torch_()
    rng = np.random.default_rng(dim + block)
    lengths = [0, 1, 70 * 16, 69 * 16 + 1, 15, 513] + [int(x) for x in rng.integers(0, 70 * 16, 14)]
    small = random_cache(rng, 30, heads, block, dim)
    width = 70 * 16 // block
    table = rng.integers(0, 30, (len(lengths), width)).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((len(lengths), 1, heads * group, dim))).to(type_of(kind)).cuda()
    whole = attend_and_check(small, q, table, lengths)
    again = attend_and_check(small, q, table, lengths)
    for a, b in zip(whole, again):
        assert torch.equal(a, b)
    wide = np.concatenate([table, np.full((len(lengths), 200), -1, np.int32)], 1)
    attend_and_check(small, q, wide, lengths)
    have = [-(-n // block) for n in lengths]
    lists = [[[[int(j) for j in rng.permutation(have[b])[:width - 1]] for _ in range(heads)]] for b in range(len(lengths))]
    attend_and_check(small, q, wide, lengths, lists)


@pytest.mark.parametrize("dim, block, heads, group, tokens, kind, tiles", [
    (128, 16, 1, 4, 1, "bf16", 64), (64, 32, 2, 8, 1, "f16", 130), (128, 64, 3, 5, 1, "bf16", 300),
    (256, 16, 2, 2, 1, "f16", 200), (128, 16, 1, 16, 1, "bf16", 1000), (64, 16, 4, 3, 2, "f16", 128),
    (256, 64, 1, 12, 1, "bf16", 96), (128, 32, 4, 24, 1, "f16", 66), (64, 64, 8, 1, 1, "bf16", 65)])
def test_attention_teams(dim, block, heads, group, tokens, kind, tiles):
    """Few longer rows, each finished by several thread blocks; some of them have nothing to do for
    a short sequence."""
    torch = torch_()
    rng = np.random.default_rng(tiles + dim)
    width = -(-tiles * 16 // block)
    lengths = [width * block, 0, width * block // 2 + 3, 5]
    small = random_cache(rng, 30, heads, block, dim)
    table = rng.integers(0, 30, (len(lengths), width)).astype(np.int32)
    table[rng.random(table.shape) < 0.03] = -1
    x = rng.standard_normal((len(lengths), tokens, heads * group, dim))
    q = torch.from_numpy(x).to(type_of(kind)).cuda()
    got = attend_and_check(small, q, table, lengths)
    again = attend_and_check(small, q, table, lengths)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    have = [-(-n // block) for n in lengths]
    lists = [[[[int(j) for j in rng.permutation(have[b])] for _ in range(heads)]
              for _ in range(tokens)] for b in range(len(lengths))]
    attend_and_check(small, q, table, lengths, lists)


@pytest.mark.parametrize("dim, block, heads, group, tokens, kind, tiles, seqs", [
    (64, 16, 2, 8, 5, "bf16", 20, 3), (128, 32, 2, 16, 4, "f16", 150, 2), (256, 16, 1, 5, 8, "bf16", 70, 4),
    (64, 64, 4, 24, 2, "f16", 40, 30), (128, 16, 1, 7, 16, "bf16", 500, 1)])
def test_attention_many_rows_without_weights(dim, block, heads, group, tokens, kind, tiles, seqs):
    """Several row tiles per key/value head, each finished by its own thread blocks."""
    torch = torch_()
    rng = np.random.default_rng(tiles + dim + seqs)
    width = -(-tiles * 16 // block)
    lengths = [width * block] + [int(x) for x in rng.integers(0, width * block, seqs - 1)]
    small = random_cache(rng, 30, heads, block, dim)
    table = rng.integers(0, 30, (seqs, width)).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((seqs, tokens, heads * group, dim))).to(type_of(kind)).cuda()
    attend_and_check(small, q, table, lengths, weights=False)


@pytest.mark.parametrize("block", [32, 64])
def test_attention_team_ends_inside_a_block(block):
    """Sequences of fewer tokens than a team has thread blocks for, and of a part of a block behind
    whole parts: the weights of the last block come from one of them."""
    torch = torch_()
    rng = np.random.default_rng(block)
    heads, dim, group = 2, 64, 4
    width = 128 * 16 // block
    lengths = [1, 17, 33, block + 1, block + 17, 3 * block + 1, width * block - 17]
    small = random_cache(rng, 30, heads, block, dim)
    table = rng.integers(0, 30, (len(lengths), width)).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((len(lengths), 1, heads * group, dim))).to(torch.bfloat16).cuda()
    for _ in range(20):
        attend_and_check(small, q, table, lengths)


def test_many_sequences_wide_tables():
    """The split over more (sequence, head) pairs than a grid's second axis holds."""
    torch = torch_()
    from hbfsim_b200 import kv_attention
    rng = np.random.default_rng(19)
    seqs, heads, dim, block = 40000, 2, 64, 16
    small = random_cache(rng, 8, heads, block, dim)
    table = np.full((seqs, 140), -1, np.int32)
    table[:, :2] = rng.integers(0, 8, (seqs, 2))
    lengths = rng.integers(0, 33, seqs)
    q = torch.from_numpy(rng.standard_normal((64, 1, 2 * heads, dim))).to(torch.bfloat16).cuda()
    q = q.repeat(seqs // 64, 1, 1, 1)
    probe = rng.integers(0, seqs, 50)
    want = ko.attention(small, q[probe].double().cpu().numpy(), table[probe], lengths[probe], dim ** -0.5)
    got = kv_attention(to_gpu(small), q, int32(table), int32(lengths), weights=True)
    assert np.abs(got.out[probe].double().cpu().numpy() - want[0]).max() <= \
        (2.0 ** -8 * np.abs(want[0]) + 2.0 ** -10 * want[3] + 2.0 ** -20).max()
    assert np.abs(got.weights[probe].double().cpu().numpy() - want[2]).max() <= 2.0 ** -17


# ---------------------------------------------------------------------------
# block lists


def assert_lists(pick, lists):
    blocks, counts = pick.blocks.cpu().numpy(), pick.counts.cpu().numpy()
    B, n, H, top = blocks.shape
    for b, t, h in itertools.product(range(B), range(n), range(H)):
        want = lists[b][t][h]
        assert counts[b, t, h] == len(want), (b, t, h)
        assert blocks[b, t, h].tolist() == want + [-1] * (top - len(want)), (b, t, h)


SELECTS = [  # dim, block, heads, group, tokens, type, lengths, top, sink, recent
    (128, 16, 2, 4, 1, "bf16", [1, 0, 16, 17, 500, 3000], 8, 1, 1),
    (64, 16, 1, 8, 3, "f16", [2, 700, 33], 5, 0, 2),
    (256, 32, 3, 16, 2, "bf16", [4000, 31], 30, 2, 3),
    (128, 64, 8, 1, 1, "f16", [64 * 40], 40, 1, 1),
    (128, 16, 8, 4, 16, "bf16", [900], 100, 1, 1),
    (64, 16, 1, 64, 1, "bf16", [16 * 2000], 1, 0, 1),
]


@pytest.mark.parametrize("dim,block,heads,group,tokens,kind,lengths,top,sink,recent", SELECTS)
def test_select(dim, block, heads, group, tokens, kind, lengths, top, sink, recent):
    torch = torch_()
    from hbfsim_b200 import kv_select
    rng = np.random.default_rng(dim + heads + group + top)
    pages = int(sum(-(-n // block) for n in lengths)) + 2
    small = random_cache(rng, min(pages, 150), heads, block, dim)
    pick = rng.integers(0, small["data"].shape[0], pages)  # many pages alike: many equal scores
    cache = {k: np.ascontiguousarray(v[pick]) for k, v in small.items()}
    table = make_table(rng, lengths, block, pages, extra=2)
    holes = rng.random(table.shape) < 0.05
    table[holes] = rng.choice([-1, pages, 1 << 30], int(holes.sum()))
    q = rng.standard_normal((len(lengths), tokens, (group + 1) * heads, dim))
    q *= 10.0 ** rng.uniform(-4, 4, q.shape[:3])[..., None]
    q = torch.from_numpy(q).to(type_of(kind)).cuda()[:, :, heads:]
    got = kv_select(to_gpu(cache), q, int32(table), int32(lengths), top, sink, recent)
    assert_lists(got, ko.select(cache, q.double().cpu().numpy(), table, lengths, top, sink, recent))


def test_select_ties_zero_and_special_queries():
    """Equal blocks are listed from the lowest index; a query of zeros ties all of them;
    NaN and infinities count as 0; the smallest and largest bfloat16."""
    torch = torch_()
    from hbfsim_b200 import kv_select
    rng = np.random.default_rng(21)
    heads, dim, block, blocks = 1, 64, 16, 3000
    cache = random_cache(rng, 1, heads, block, dim)
    cache = {k: np.repeat(v, 2, 0) for k, v in cache.items()}
    table = rng.integers(0, 2, (5, blocks)).astype(np.int32)
    q = rng.standard_normal((5, 1, 2, dim))
    q[1] = 0
    q[2, 0, 0, ::3] = np.nan
    q[2, 0, 1, ::5] = np.inf
    q[3] *= 1e-40
    q[4] *= 3e38 / np.abs(q[4]).max()
    q = torch.from_numpy(q).to(torch.bfloat16).cuda()
    lengths = [blocks * block] * 5
    got = kv_select(to_gpu(cache), q, int32(table), int32(lengths), 700, 2, 2)
    assert_lists(got, ko.select(cache, q.double().cpu().numpy(), table, lengths, 700, 2, 2))


# ---------------------------------------------------------------------------
# eviction

EVICTS = [  # block, heads, lengths, keep, sink, recent, decay
    (16, 1, [1, 0, 16, 17, 100], 2, 1, 1, 0),
    (16, 8, [3000, 16 * 60, 500], 60, 1, 1, 8),
    (32, 3, [32 * 2500, 32 * 1024, 32 * 1025 - 31], 1024, 4, 16, 1),
    (64, 2, [64 * 300], 1, 0, 1, 63),
    (16, 4, [16 * 5000], 4999, 0, 4999, 0),
]


@pytest.mark.parametrize("block,heads,lengths,keep,sink,recent,decay", EVICTS)
@pytest.mark.parametrize("levels", [0, 3])
def test_evict(block, heads, lengths, keep, sink, recent, decay, levels):
    """levels > 0: scores of few values, so that ties decide."""
    torch = torch_()
    from hbfsim_b200 import kv_evict
    rng = np.random.default_rng(block + heads + keep + levels)
    B = len(lengths)
    pages = int(sum(-(-n // block) for n in lengths)) + 2
    table = make_table(rng, lengths, block, pages, extra=5)
    width = table.shape[1]
    if levels:
        score = rng.integers(-levels, levels, (B, width))
        weights = rng.integers(0, levels, (B, heads, width)).astype(np.float32) * 2.0 ** -30
    else:
        score = rng.integers(-(1 << 40), 1 << 40, (B, width))
        weights = (rng.random((B, heads, width)) ** 8).astype(np.float32)
        for i, odd in enumerate((np.nan, -1.0, np.inf, 1e30, -np.inf, 2.0 ** 20)):
            weights[rng.integers(B), rng.integers(heads), rng.integers(width)] = odd
    got = kv_evict(torch.from_numpy(score).cuda(), torch.from_numpy(weights).cuda(), int32(table),
                   int32(lengths), keep, block, sink, recent, decay)
    want = ko.evict(score, weights, table, lengths, keep, block, sink, recent, decay)
    for a, b, name in zip(got, want, got._fields):
        assert np.array_equal(a.cpu().numpy(), b), name


# ---------------------------------------------------------------------------
# together


def test_decode_steps_and_their_reads(tmp_path):
    """Prompt, then decode steps of select, attend and evict on one cache that the simulator
    times: what leaves is freed, what is read is listed, and the simulator models every read."""
    torch = torch_()
    from helpers import Setup, make_context
    from hbfsim_b200 import KvCache, kv_append, kv_attention, kv_block_reads, kv_evict, kv_select
    from hbfsim_b200 import workloads as wl
    rng = np.random.default_rng(31)
    heads, group, dim, block, seqs, keep = 2, 4, 128, 16, 3, 6
    pages, width = 60, 12
    setup = Setup(profile=wl.c0_profile(), model=3)
    setup.ranges = [(wl.RANGE_BASE, 1 << 30, 1, 3)]
    ctx = make_context(setup, str(tmp_path))
    gpu = KvCache.empty(pages, heads, dim, block)
    cache = from_gpu(gpu)
    prompt = np.array([150, 33, 5])
    free = list(rng.permutation(pages))
    table = np.full((seqs, width), -1, np.int32)
    lengths = prompt.copy()
    for b in range(seqs):
        for j in range(-(-prompt[b] // block)):
            table[b, j] = free.pop()
    offsets = np.concatenate([[0], np.cumsum(prompt)])

    def new(shape):
        return torch.from_numpy(rng.standard_normal(shape)).to(torch.bfloat16).cuda()

    k, v = new((offsets[-1], heads, dim)), new((offsets[-1], heads, dim))
    kv_append(gpu, k, v, int32(table), int32([0] * seqs), offsets=int32(offsets))
    ko.append(cache, k.double().cpu().numpy(), v.double().cpu().numpy(), table, [0] * seqs, offsets)
    score = torch.zeros((seqs, width), dtype=torch.int64, device="cuda")
    clock = 0
    for _ in range(20):
        for b in range(seqs):
            if lengths[b] % block == 0:
                table[b, lengths[b] // block] = free.pop()
        q = new((seqs, 1, heads * group, dim))
        k, v = new((seqs, 1, heads, dim)), new((seqs, 1, heads, dim))
        kv_append(gpu, k, v, int32(table), int32(lengths))
        flat = [t.double().cpu().numpy().reshape(seqs, heads, dim) for t in (k, v)]
        ko.append(cache, *flat, table, lengths, np.arange(seqs + 1))
        lengths = lengths + 1
        same_cache(gpu, cache)
        pick = kv_select(gpu, q, int32(table), int32(lengths), top=4)
        lists = ko.select(cache, q.double().cpu().numpy(), table, lengths, 4, 1, 1)
        assert_lists(pick, lists)
        got = attend_and_check(cache, q, table, lengths, lists, gpu=gpu)
        address, nbytes, op = kv_block_reads(gpu, int32(table), pick.blocks, pick.counts,
                                             wl.RANGE_BASE)
        flat_lists = [(table[b, j], h) for b in range(seqs) for h in range(heads)
                      for j in lists[b][0][h]]
        assert ((address.cpu().numpy() - wl.RANGE_BASE) // 4096).tolist() == \
            [p * heads + h for p, h in flat_lists]
        arrival = torch.full_like(address, clock)
        timed = ctx.submit(address, nbytes, op, arrival)
        assert (timed.status == 1).all()
        clock = int(timed.done_ns.max())
        rest = kv_evict(score, got.weights, int32(table), int32(lengths), keep, block)
        freed = rest.freed.cpu().numpy()
        for b in range(seqs):
            free += freed[b, :int(rest.freed_counts[b])].tolist()
        score, table, lengths = rest.score, rest.table.cpu().numpy(), rest.lengths.cpu().numpy()
        assert (-(-lengths // block) <= keep).all()
    ctx.close()


@pytest.mark.parametrize("seqs,blocks,keep,kind", [(1, 3000, 2000, "equal"), (1, 20000, 100, "octaves"),
                                                   (2, 9000, 8999, "zeros"), (1, 5000, 40, "equal"),
                                                   (1, 250000, 1000, "octaves")])
def test_evict_long_rows(seqs, blocks, keep, kind):
    """Rows that several thread blocks share, and one that none can hold: all scores equal,
    scores of many orders, mostly zeros."""
    torch = torch_()
    from hbfsim_b200 import kv_evict
    rng = np.random.default_rng(blocks)
    table = rng.permutation(seqs * blocks).reshape(seqs, blocks).astype(np.int32)
    lengths = [blocks * 16 - 5 * b for b in range(seqs)]
    weights = np.zeros((seqs, 2, blocks), np.float32)
    if kind == "equal":
        score = np.full((seqs, blocks), 77, np.int64)
    elif kind == "zeros":
        score = np.where(rng.random((seqs, blocks)) < 0.001, 5, 0)
    else:
        score = (2.0 ** rng.uniform(0, 50, (seqs, blocks))).astype(np.int64)
        weights = (2.0 ** rng.uniform(-30, 5, weights.shape)).astype(np.float32)
    got = kv_evict(torch.from_numpy(score).cuda(), torch.from_numpy(weights).cuda(), int32(table),
                   int32(lengths), keep)
    want = ko.evict(score, weights, table, lengths, keep, 16, 1, 1, 0)
    for a, b, name in zip(got, want, got._fields):
        assert np.array_equal(a.cpu().numpy(), b), name


@pytest.mark.parametrize("blocks,top,heads", [(6000, 37, 2), (40000, 5000, 1), (300000, 64, 1)])
def test_select_long_rows(blocks, top, heads):
    """Rows that several thread blocks share, and one that none can hold; few distinct pages, so
    that ties decide at the end of the list."""
    torch = torch_()
    from hbfsim_b200 import kv_select
    rng = np.random.default_rng(blocks)
    dim, block = 64, 16
    cache = random_cache(rng, 300, heads, block, dim)
    table = rng.integers(0, 300, (1, blocks)).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((1, 1, heads, dim))).to(torch.bfloat16).cuda()
    got = kv_select(to_gpu(cache), q, int32(table), int32([blocks * block - 3]), top)
    assert_lists(got, ko.select(cache, q.double().cpu().numpy(), table, [blocks * block - 3], top, 1, 1))


@pytest.mark.parametrize("blocks, top, recent", [
    (511, 40, 1), (512, 512, 3), (513, 512, 1), (2048, 1, 1), (2049, 2000, 900), (4096, 77, 70), (4097, 4000, 1),
    (8192, 256, 1), (8193, 8192, 5000), (16384, 300, 300), (16385, 16385, 2)])
def test_select_widths(blocks, top, recent):
    """Tables at the widths where the selection changes its form; rows from empty to full, with few
    distinct pages (ties), and lists from always listed blocks alone to every block."""
    torch = torch_()
    from hbfsim_b200 import kv_select
    rng = np.random.default_rng(blocks + top)
    heads, dim, block, tokens = 2, 64, 16, 2
    cache = random_cache(rng, 40, heads, block, dim)
    lengths = [blocks * block, 0, 1, blocks * block // 2 + 5, min(blocks * block, (top + 1) * block)]
    table = rng.integers(0, 40, (len(lengths), blocks)).astype(np.int32)
    table[rng.random(table.shape) < 0.02] = -1
    q = torch.from_numpy(rng.standard_normal((len(lengths), tokens, 3 * heads, dim))).to(torch.bfloat16).cuda()
    got = kv_select(to_gpu(cache), q, int32(table), int32(lengths), top, 0, recent)
    assert_lists(got, ko.select(cache, q.double().cpu().numpy(), table, lengths, top, 0, recent))


def test_example(capsys):
    """The example: fewer reads and less simulated time for the lists than for every block, and
    what is evicted is what goes beyond `keep`."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "kv_decode.py"
    spec = importlib.util.spec_from_file_location("kv_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.main(["--seqs", "3", "--context", "500", "--steps", "20", "--top", "6", "--keep", "20"])
    assert "listed_reads" in capsys.readouterr().out
    assert got["listed_reads"] == 3 * 20 * 8 * 6
    # 32 blocks after the first token; 20 stay, then one leaves for each that begins
    begun = [-(-(500 + 20) // 16) - 32] * 3
    assert got["evicted_blocks"] == sum(12 + n for n in begun)
    assert got["every_reads"] > 3 * got["listed_reads"]
    assert got["every_us_per_step"] > got["listed_us_per_step"] > 0


def test_evict_into_memory_between_the_inputs():
    """Outputs beside the inputs in one allocation, between the rows of a strided table too."""
    import ctypes
    torch = torch_()
    from hbfsim_b200 import _lib
    rng = np.random.default_rng(41)
    seqs, heads, width, keep = 3, 2, 40, 9
    pool = torch.zeros(1 << 14, dtype=torch.int32, device="cuda")
    at = dict(table=0, table_out=40, freed=160, lengths=300, lengths_out=303, freed_counts=306, weights=400,
              score=1000, score_out=1000 + 2 * seqs * width)
    stride = 4096  # rows of the table, the outputs between the first two

    def put(name, x):
        x = torch.from_numpy(np.ascontiguousarray(x)).cuda().view(torch.int32).flatten()
        pool[at[name]:at[name] + x.numel()] = x

    table = rng.permutation(seqs * width).reshape(seqs, width).astype(np.int32)
    for b in range(seqs):
        pool[b * stride:b * stride + width] = torch.from_numpy(table[b]).cuda()
    score = rng.integers(0, 1 << 40, (seqs, width))
    weights = rng.random((seqs, heads, width)).astype(np.float32)
    lengths = np.array([40 * 16, 100, 39 * 16 + 1], np.int32)
    put("score", score)
    put("weights", weights)
    put("lengths", lengths)
    where = {k: pool.data_ptr() + 4 * v for k, v in at.items()}
    batch = _lib.KvEvictBatchV1(struct_size=ctypes.sizeof(_lib.KvEvictBatchV1), version=1, seqs=seqs, kv_heads=heads,
                                width=width, block_tokens=16, keep=keep, sink=1, recent=1, decay=4,
                                table_stride=stride, **where)
    torch.cuda.synchronize()
    assert _lib.load().hbfsim_kv_evict_v1(ctypes.byref(batch), None) == 0
    torch.cuda.synchronize()
    want = ko.evict(score, weights, table, lengths, keep, 16, 1, 1, 4)
    got = pool.cpu().numpy()
    for name, x in zip(("score_out", "table_out", "lengths_out", "freed", "freed_counts"), want):
        flat = np.ascontiguousarray(x).view(np.int32).ravel()
        assert np.array_equal(got[at[name]:at[name] + flat.size], flat), name


@pytest.mark.parametrize("name", ["top", "sink", "recent", "keep", "block_tokens", "esink", "erecent", "decay"])
@pytest.mark.parametrize("value", [-1, 1 << 32, (1 << 32) + 1, 1 << 70])
def test_counts_that_do_not_fit_are_refused(name, value):
    """A count past 32 bits is not taken for what remains of it."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_evict, kv_select
    table = torch.zeros((1, 3), dtype=torch.int32, device="cuda")
    if name in ("top", "sink", "recent"):
        q = torch.ones((1, 1, 2, 64), dtype=torch.float16, device="cuda")
        with pytest.raises(ValueError):
            kv_select(KvCache.empty(2, 2, 64), q, table, int32([40]), **{"top": 3, name: value})
    else:
        score = torch.zeros((1, 3), dtype=torch.int64, device="cuda")
        with pytest.raises(ValueError):
            kv_evict(score, torch.zeros((1, 1, 3), device="cuda"), table, int32([40]),
                     **{"keep": 2, name.lstrip("e"): value})


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), 10 ** 400])
def test_scales_that_do_not_fit_are_refused(scale):
    torch = torch_()
    from hbfsim_b200 import HbfsimError, KvCache, kv_attention
    q = torch.ones((1, 1, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises((ValueError, HbfsimError)):
        kv_attention(KvCache.empty(2, 2, 64), q, torch.zeros((1, 3), dtype=torch.int32, device="cuda"), int32([40]),
                     scale=scale)


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_gradients_are_refused_not_dropped(which):
    """No operator here has a backward pass: a tensor that asks for one raises, unless gradients
    are off."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_append, kv_attention, kv_select
    gpu = KvCache.empty(4, 2, 64)
    table = torch.zeros((1, 3), dtype=torch.int32, device="cuda")
    make = lambda heads, name: torch.ones((1, 1, heads, 64), dtype=torch.float16, device="cuda",  # noqa: E731
                                          requires_grad=which == name)
    q, k, v = make(4, "q"), make(2, "k"), make(2, "v")

    def call():
        kv_append(gpu, k, v, table, int32([0]))
        return kv_attention(gpu, q * 1, table, int32([1]))

    with pytest.raises(ValueError, match="gradient"):
        call()
    kv_select(gpu, q, table, int32([1]), top=2)  # block lists have no gradient
    with torch.no_grad():
        want = call()
    with torch.inference_mode():
        assert torch.equal(call().out, want.out)
    q, k, v = q.detach(), k.detach(), v.detach()
    assert torch.equal(call().out, want.out)


STALE_ERROR = """
import ctypes
import torch
from hbfsim_b200 import HbfsimError, KvCache, kv_append, kv_evict

gpu = KvCache.empty(4, 2, 64)
table = torch.zeros((1, 3), dtype=torch.int32, device="cuda")
lengths = torch.tensor([20], dtype=torch.int32, device="cuda")
k = torch.ones((1, 1, 2, 64), dtype=torch.float16, device="cuda")
score, weights = torch.zeros((1, 3), dtype=torch.int64, device="cuda"), torch.zeros((1, 2, 3), device="cuda")
kv_append(gpu, k, k, table, lengths)
kv_evict(score, weights, table, lengths, keep=2)
torch.cuda.synchronize()
runtime = ctypes.CDLL("libcudart.so.12")  # the one that torch has loaded
handle = ctypes.c_void_p()
assert runtime.cudaStreamCreate(ctypes.byref(handle)) == 0  # ordered with the legacy stream
assert runtime.cudaStreamBeginCapture(handle, 0) == 0
# a launch into the legacy stream is an error as long as the capture lasts, and ends it
refused = False
try:
    kv_evict(score, weights, table, lengths, keep=2)
except HbfsimError:
    refused = True
graph = ctypes.c_void_p()
assert runtime.cudaStreamEndCapture(handle, ctypes.byref(graph)) != 0 and refused
runtime.cudaGetLastError()
kv_append(gpu, k, k, table, lengths)  # its launch succeeds: no error of the call before
torch.cuda.synchronize()
print("fine")
"""


def test_an_error_is_reported_once():
    """A launch that failed does not make the next call fail."""
    import os
    import subprocess
    import sys
    from pathlib import Path
    run = subprocess.run([sys.executable, "-c", STALE_ERROR], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parent.parent, env=dict(os.environ))
    assert run.returncode == 0 and "fine" in run.stdout, run.stderr[-2000:]
