"""The forms of the operators around the attention that large calls take: lists of many moves, rotary
appends with many tokens and heads, and page operators at the sizes where their form changes.  Equal to
the definitions, as in the tests of small calls.  Which form a call takes follows from its sizes and the
number of SMs; sizes here follow from it too."""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import int32, make_table, same_cache, to_gpu, torch_, type_of
from test_kv_pages_gpu import pool, resize_and_check, same
from test_kv_rotary_gpu import plain, rotary_of, same_queries

pytestmark = pytest.mark.gpu


def sms():
    return torch_().cuda.get_device_properties(0).multi_processor_count


# ---------------------------------------------------------------------------
# copies: lists of more than 512 pieces (16 KB of a page) to an SM go by several moves to a thread block


@pytest.mark.parametrize("heads,dim,pages", [(1, 64, 50000), (5, 128, 4000)])  # one piece to a page, and two
@pytest.mark.parametrize("group,rest", [(2, 1), (3, 76), (7, 0), (32, 5), (32, 1 << 20)])
def test_copy_long_lists(heads, dim, pages, group, rest):
    """Mostly empty lists, as a compaction gives them, with moves on both sides of the groups' borders and
    in the last group; entries that leave either pool among them."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_copy
    block, page_bytes = 16, heads * 2 * 16 * dim
    pieces = -(-page_bytes // 16384)
    count = -(-512 * sms() * (group - 1) // pieces) + rest
    assert min(32, count * pieces // (512 * sms()) + 1) == group
    gen = torch.Generator(device="cuda").manual_seed(group + rest + heads)
    gpu = KvCache.empty(pages, heads, dim, block)
    of = [gpu.data.view(torch.uint8), gpu.scale, gpu.bounds]
    of[0].copy_(torch.randint(0, 256, of[0].shape, generator=gen, device="cuda"))
    of[1].copy_(torch.rand(of[1].shape, generator=gen, device="cuda"))
    of[2].copy_(torch.randint(-112, 113, of[2].shape, generator=gen, device="cuda"))
    want = [x.clone() for x in of]
    rng = np.random.default_rng(group + rest)
    order = rng.permutation(pages)
    places = rng.permutation(count)[:pages // 3]
    edges = np.concatenate([group * np.array([1, 2, 9, 31]) + d for d in (-1, 0)])
    places = np.unique(np.concatenate([places, edges, [0, count - 1, count - 2, count - group]]))[:pages // 2]
    src, dst = np.full(count, -1, np.int32), np.full(count, -1, np.int32)
    src[places], dst[places] = order[:len(places)], order[-len(places):]
    assert src[count - 1] >= 0 and src[0] >= 0
    bad = places[5::9]
    src[bad[::3]], dst[bad[1::3]], src[bad[2::3]] = -7, pages, 2 ** 31 - 1
    empty = np.setdiff1d(np.arange(0, count, 101), places)
    src[empty] = 1  # nowhere to go
    kv_copy(gpu, int32(src), int32(dst))
    real = (src >= 0) & (src < pages) & (dst >= 0) & (dst < pages)
    a, b = (torch.from_numpy(x[real].astype(np.int64)).cuda() for x in (src, dst))
    for got, w in zip(of, want):
        w[b] = w[a]
        assert torch.equal(got, w)


# ---------------------------------------------------------------------------
# rotary appends


def rotary_form(tokens, seqs, heads, block):
    """Tokens of a chunk, heads' keys that a thread block takes one after the other."""
    chunk = 1
    while chunk < (32 if block == 16 else 16) and tokens * heads * 2 > chunk * 16 * sms():
        chunk *= 2
    teams = 64 // block
    return chunk, 8 if (tokens // block + seqs) * heads > 12 * teams * sms() else teams


ROTARY = [  # dim, block, heads, type, share of the channels, neighbours, odd strides, seqs, eight heads in turn
    (64, 16, 64, "bf16", 1, False, False, 30, True),
    (128, 16, 20, "bf16", 1, False, False, 60, True),
    (128, 16, 12, "f16", 2, False, True, 60, True),
    (256, 16, 9, "f16", 1, True, False, 150, True),
    (64, 32, 20, "f16", 2, True, False, 50, True),
    (128, 32, 20, "bf16", 1, True, False, 40, True),
    (256, 32, 9, "bf16", 1, False, False, 100, True),
    (64, 64, 12, "bf16", 1, False, True, 30, True),
    (128, 64, 20, "bf16", 1, False, False, 20, True),
    (256, 64, 9, "f16", 2, False, False, 60, True),
    (128, 16, 2, "bf16", 1, False, False, 7, False),
    (256, 16, 2, "bf16", 1, False, False, 9, False),
    (128, 32, 2, "f16", 1, False, False, 5, False),
    (128, 64, 1, "bf16", 4, True, False, 3, False),
    (256, 64, 1, "bf16", 1, False, False, 4, False),
]


@pytest.mark.parametrize("dim,block,heads,kind,part,neighbours,odd,seqs,turns", ROTARY)
def test_rotary_append_of_many_tokens(dim, block, heads, kind, part, neighbours, odd, seqs, turns):
    """Chunks of as many tokens as there are, cosines of whole chunks and the blocks behind them in shared
    memory, heads one after the other (the last group of them not full); sequences that begin and end
    inside blocks, of one token and of none."""
    torch = torch_()
    from hbfsim_b200 import kv_append_rotary
    rng = np.random.default_rng(dim + block + heads)
    most = 32 if block == 16 else 16
    tokens = max(8 * most * sms() // heads + 200,
                 (12 * (64 // block) * sms() // heads - seqs + 2) * block if turns else 0)
    chunk, by = rotary_form(tokens, seqs, heads, block)
    assert chunk == most and (by == 8) == turns
    weight = rng.random(seqs) + 0.05
    weight[1] = 0
    count = np.floor((tokens - 1) * weight / weight.sum()).astype(np.int64)
    count[2] = 1
    count[0] += tokens - count.sum()
    start = rng.integers(0, 3 * block, seqs).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    blocks = -(-(start + count) // block)
    pages = int(blocks.sum()) + 2
    shape = (pages, heads, 2)
    data = rng.integers(0, 256, shape + (block, dim), np.uint8)
    data[data % 128 == 127] = 0  # no NaN
    cache = dict(data=data, scale=2.0 ** rng.integers(-14, 4, shape), bounds=np.zeros(shape + (dim,), np.int8))
    table = make_table(rng, start + count, block, pages)
    x = rng.standard_normal((tokens, 3 * heads, dim + odd), np.float32) * 10.0 ** rng.uniform(-3, 3, (tokens, 1, 1))
    qkv = torch.from_numpy(x).to(type_of(kind)).cuda()[..., odd:]
    q, k, v = qkv[:, :heads], qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    pairs = dim // 2 // part
    positions = rng.integers(0, 9000, (3, tokens)).astype(np.int32)
    freq, axis = 1e4 ** (-np.arange(pairs) / pairs), np.arange(pairs) % 3
    gpu = to_gpu(cache)
    got = kv_append_rotary(gpu, q, k, v, int32(table), int32(start), int32(positions), rotary_of(freq, axis, neighbours),
                           offsets=int32(offsets))
    same_queries(got, q, positions, freq, axis, neighbours)
    turned = ko.rotate(plain(k), positions, freq, axis, neighbours).astype(np.float64)
    ko.append(cache, turned, v.double().cpu().numpy(), table, start, offsets)
    same_cache(gpu, cache)


# ---------------------------------------------------------------------------
# pages: a resize takes one cluster up to 262,144 counts and 131,072 entries (of 1, 2, 4 or 8 thread
# blocks: 16,384 counts, 16,384 entries and 32 runs of 512 entries each), a launch to a pass beyond; a
# compaction one thread block up to 8,192 of both


@pytest.mark.parametrize("seqs,width,pages", [
    (4, 16, 262144), (4, 16, 262145), (64, 2048, 3000), (3, 43691, 9000), (9, 1820, 16384), (9, 1821, 16385),
    (32, 512, 900), (33, 512, 900), (32, 513, 900), (700, 20, 9000), (4096, 32, 90000), (20000, 6, 50000)])
def test_resize_where_its_form_changes(seqs, width, pages):
    rng = np.random.default_rng(seqs + width + pages)
    refs, table, lengths = pool(rng, seqs, width, pages, 16)
    kind = rng.integers(0, 5, seqs)
    want = np.select([kind == 0, kind == 1, kind == 2, kind == 3],
                     [0 * lengths, lengths // 2, lengths, lengths + 1], lengths + rng.integers(0, 200, seqs)).astype(np.int32)
    resize_and_check(refs, table, lengths, want)


@pytest.mark.parametrize("pages,seqs,width", [(8192, 4, 2048), (8193, 4, 2048), (8192, 1, 8193), (100, 8193, 1), (9000, 2, 3)])
def test_compact_where_its_form_changes(pages, seqs, width):
    from hbfsim_b200 import kv_compact
    rng = np.random.default_rng(pages + width)
    refs = np.where(rng.random(pages) < 0.6, rng.integers(1, 5, pages), 0).astype(np.int32)
    table = rng.integers(-3, pages + 3, (seqs, width)).astype(np.int32)
    want = ko.compact(refs, table)
    r, t = int32(refs), int32(table)
    same(kv_compact(r, t), want)
    same(kv_compact(r, t, inplace=True), want)


@pytest.mark.parametrize("seqs,width,rows", [(2000, 40, 2000), (3, 16385, 700), (5000, 2, 300)])
def test_fork_of_many_rows(seqs, width, rows):
    from hbfsim_b200 import kv_fork
    rng = np.random.default_rng(seqs + rows)
    refs, table, lengths = pool(rng, seqs, width, 60000, 16)
    parents = rng.integers(-1, seqs + 1, rows).astype(np.int32)
    want = ko.fork(refs, table, lengths, parents, 16)
    for inplace in (False, True):
        same(kv_fork(int32(refs), int32(table), int32(lengths), int32(parents), inplace=inplace), want)
