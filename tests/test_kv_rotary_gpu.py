"""kv_append_rotary against its definition (oracle/kv_oracle.py): equal in every value.

Angles are products in 64 bits; sines and cosines are right to 1e-14 and rounded to 32 bits (half a
step: 6e-8 of 1), so they differ from the oracle's only where a value lies that near to the middle
between two 32-bit numbers: once in a million, and in none of the inputs here.  Everything after
them is single products and sums rounded to 32 bits, and the roundings to the output's type and to
e4m3, which are parts of the definition.  One test holds the queries to the formula in 64 bits:
2^-24 of |x| + |y| for the rounded cosines, as much again for the products and the sum, and half a
step of the type.
"""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import from_gpu, int32, make_table, random_cache, same_cache, to_gpu, torch_, type_of

pytestmark = pytest.mark.gpu


def rotary_of(freq, axis, neighbours):
    torch = torch_()
    from hbfsim_b200 import KvRotary
    return KvRotary(torch.from_numpy(np.asarray(freq, np.float64)).cuda(),
                    torch.from_numpy(np.asarray(axis, np.uint8)).cuda(), neighbours)


def plain(t):
    """As float32 [tokens, heads, dim] on the host."""
    return t.float().cpu().numpy().reshape((-1,) + tuple(t.shape[-2:]))


def same_queries(got, q, positions, freq, axis, neighbours):
    torch = torch_()
    want = torch.from_numpy(ko.rotate(plain(q), positions, freq, axis, neighbours)).to(q.dtype).float()
    assert got.dtype == q.dtype and got.shape == q.shape and got.is_contiguous()
    assert np.array_equal(plain(got), want.numpy(), equal_nan=True), "queries"


CASES = [  # dim, block, heads, group, type, pairs, axes, neighbours, (start, new) per sequence
    (128, 16, 2, 4, "bf16", 64, 3, False, [(0, 1)]),
    (128, 16, 1, 1, "bf16", 64, 1, False, [(15, 1), (16, 1), (17, 1), (0, 0)]),
    (128, 16, 8, 4, "bf16", 64, 3, False, [(5, 40), (0, 16), (31, 1), (16, 17), (7, 0), (100, 3)]),
    (128, 16, 2, 7, "f16", 32, 4, False, [(0, 33), (14, 5)]),
    (128, 32, 3, 2, "f16", 4, 2, False, [(30, 5), (0, 70)]),
    (128, 64, 1, 9, "bf16", 64, 3, True, [(63, 2), (1, 200)]),
    (64, 16, 2, 8, "f16", 32, 1, False, [(0, 50)]),
    (64, 64, 2, 3, "bf16", 16, 3, True, [(60, 70), (0, 64)]),
    (64, 32, 1, 1, "f16", 2, 1, True, [(0, 32), (1, 32), (2, 100)]),
    (256, 16, 2, 2, "bf16", 128, 3, False, [(0, 17), (16, 16), (9, 1)]),
    (256, 32, 1, 8, "f16", 64, 1, False, [(30, 5), (0, 33), (64, 64)]),
    (256, 64, 1, 1, "bf16", 128, 4, True, [(0, 64), (63, 66)]),
    (256, 64, 3, 1, "f16", 8, 2, False, [(0, 150)]),
]


@pytest.mark.parametrize("dim,block,heads,group,kind,pairs,axes,neighbours,what", CASES)
def test_append_rotary(dim, block, heads, group, kind, pairs, axes, neighbours, what):
    torch = torch_()
    from hbfsim_b200 import kv_append_rotary
    rng = np.random.default_rng(dim + block + heads + pairs)
    start = np.array([s for s, _ in what], np.int32)
    count = np.array([n for _, n in what])
    offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    lengths = start + count
    pages = int(sum(-(-n // block) for n in lengths)) + 2
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, lengths, block, pages, extra=1)
    total, rows = int(offsets[-1]), (group + 2) * heads
    x = rng.standard_normal((total, rows, dim)) * 10.0 ** rng.uniform(-3, 3, (total, rows, 1))
    qkv = torch.from_numpy(x).to(type_of(kind)).cuda()
    q, k, v = qkv[:, :group * heads], qkv[:, group * heads:-heads], qkv[:, -heads:]
    positions = rng.integers(0, 300000, (axes, total)).astype(np.int32)
    positions[:, 0] = 0
    positions[0, -1] = -7  # before the beginning
    freq = 1e4 ** (-np.arange(pairs) / pairs)
    axis = rng.integers(0, axes, pairs)
    gpu = to_gpu(cache)
    for _ in range(2):  # the same tokens again leave everything as it is
        got = kv_append_rotary(gpu, q, k, v, int32(table), int32(start), int32(positions),
                               rotary_of(freq, axis, neighbours), offsets=int32(offsets))
        same_queries(got, q, positions, freq, axis, neighbours)
        turned = ko.rotate(plain(k), positions, freq, axis, neighbours).astype(np.float64)
        ko.append(cache, turned, v.double().cpu().numpy(), table, start, offsets)
        same_cache(gpu, cache)


@pytest.mark.parametrize("seqs,tokens,heads", [(700, 1, 1), (3, 1500, 2), (41, 63, 8), (5, 7, 64)])
def test_many_tokens(seqs, tokens, heads):
    """From one token to a thread block to sixteen, with sequences that end inside a chunk."""
    torch = torch_()
    from hbfsim_b200 import kv_append_rotary
    rng = np.random.default_rng(seqs)
    dim, block, pairs = 64, 16, 32
    start = rng.integers(0, 40, seqs).astype(np.int32)
    count = np.full(seqs, 1) if tokens == 1 else rng.integers(0, 2 * tokens, seqs)
    offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    pages = int((-(-(start + count) // block)).sum()) + 2
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, start + count, block, pages)
    qkv = torch.from_numpy(rng.standard_normal((int(offsets[-1]), 4 * heads, dim))).to(torch.bfloat16).cuda()
    q, k, v = qkv[:, :2 * heads], qkv[:, 2 * heads:3 * heads], qkv[:, 3 * heads:]
    positions = rng.integers(0, 5000, (3, int(offsets[-1]))).astype(np.int32)
    freq, axis = 1e4 ** (-np.arange(pairs) / pairs), np.arange(pairs) % 3
    gpu = to_gpu(cache)
    got = kv_append_rotary(gpu, q, k, v, int32(table), int32(start), int32(positions),
                           rotary_of(freq, axis, False), offsets=int32(offsets))
    same_queries(got, q, positions, freq, axis, False)
    turned = ko.rotate(plain(k), positions, freq, axis, False).astype(np.float64)
    ko.append(cache, turned, v.double().cpu().numpy(), table, start, offsets)
    same_cache(gpu, cache)


@pytest.mark.parametrize("neighbours", [False, True])
def test_uniform_odd_strides_and_one_axis(neighbours):
    """[seqs, n, heads, dim] without offsets; rows that start at odd elements; positions without an
    axis of their own; no queries."""
    torch = torch_()
    from hbfsim_b200 import KvRotary, kv_append_rotary
    rng = np.random.default_rng(5)
    heads, dim, block, seqs, n = 2, 64, 16, 3, 18
    start = np.array([14, 0, 29], np.int32)
    cache = random_cache(rng, 12, heads, block, dim)
    table = make_table(rng, start + n, block, 12)
    wide = torch.from_numpy(rng.standard_normal((seqs * n, heads, dim + 3))).to(torch.bfloat16).cuda()
    k = wide[:, :, 1:dim + 1].unflatten(0, (seqs, n))
    v = wide[:, :, 3:].unflatten(0, (seqs, n))
    q = wide[:, :, 2:dim + 2].unflatten(0, (seqs, n)).transpose(0, 1).contiguous().transpose(0, 1)
    places = start[:, None] + np.arange(n, dtype=np.int32)
    rotary = KvRotary.of(dim, base=500.0, neighbours=neighbours)
    freq, axis = rotary.freq.cpu().numpy(), rotary.axis.cpu().numpy()
    assert np.allclose(freq, 500.0 ** (-np.arange(32) / 32), rtol=1e-15)
    gpu = to_gpu(cache)
    got = kv_append_rotary(gpu, q, k, v, int32(table), int32(start), int32(places), rotary)
    same_queries(got, q, places.reshape(1, -1), freq, axis, neighbours)
    turned = ko.rotate(plain(k), places.reshape(1, -1), freq, axis, neighbours).astype(np.float64)
    ko.append(cache, turned, v.double().cpu().numpy().reshape(seqs * n, heads, dim), table, start,
              np.arange(seqs + 1) * n)
    same_cache(gpu, cache)
    # keys alone, positions as a strided view of [seqs, n, axes]
    stacked = int32(np.stack([places, places], -1)).permute(2, 0, 1)
    assert kv_append_rotary(gpu, None, k, v, int32(table), int32(start), stacked, rotary) is None
    same_cache(gpu, cache)


def test_queries_against_the_formula():
    torch = torch_()
    from hbfsim_b200 import KvCache, KvRotary, kv_append_rotary
    rng = np.random.default_rng(8)
    tokens, heads, dim = 200, 4, 128
    rotary = KvRotary.of(dim, base=1e6, sections=(16, 24, 24))
    freq, axis = rotary.freq.cpu().numpy(), rotary.axis.cpu().numpy()
    assert axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    positions = rng.integers(0, 1 << 20, (3, tokens)).astype(np.int32)
    for kind in ("bf16", "f16"):
        q = torch.from_numpy(rng.standard_normal((tokens, heads, dim))).to(type_of(kind)).cuda()
        kv = q[:, :1]
        got = kv_append_rotary(KvCache.empty(1, 1, dim), q, kv, kv, int32(np.full((1, 1), -1)), int32([0]),
                               int32(positions), rotary, offsets=int32([0, tokens]))
        x, y = (q.double().cpu().numpy()[..., i] for i in (slice(0, 64), slice(64, 128)))
        a = (positions[axis].astype(np.float64).T * freq)[:, None]
        want = np.concatenate([x * np.cos(a) - y * np.sin(a), x * np.sin(a) + y * np.cos(a)], -1)
        size = np.concatenate([np.abs(x) + np.abs(y)] * 2, -1)
        off = np.abs(got.double().cpu().numpy() - want)
        unit = torch.finfo(q.dtype).eps / 2
        assert (off <= unit * np.abs(want) + (1 + unit) * 3 * 2.0 ** -24 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("size", [1e5, 4e9, 1e18])
def test_angles_of_every_size(size):
    """Frequencies far above 1: angles past the first reduction's range too; and ones near multiples
    of a quarter turn, where the sine or cosine is small."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_append_rotary
    rng = np.random.default_rng(9)
    tokens, pairs = 400, 32
    positions = rng.integers(-(1 << 31), 1 << 31, (1, tokens)).astype(np.int32)
    positions[0, :40] = np.arange(40) - 20
    freq = size / 2.0 ** 31 * rng.uniform(0.5, 1, pairs)
    freq[:4] = np.pi / 2 * np.array([1, 2, 1001, 65536])
    axis = np.zeros(pairs, int)
    q = torch.from_numpy(rng.standard_normal((tokens, 2, 64))).to(torch.bfloat16).cuda()
    kv = q[:, :1]
    got = kv_append_rotary(KvCache.empty(1, 1, 64), q, kv, kv, int32(np.full((1, 1), -1)), int32([0]),
                           int32(positions), rotary_of(freq, axis, False), offsets=int32([0, tokens]))
    same_queries(got, q, positions, freq, axis, False)


def test_special_values_and_absent_blocks():
    """Infinities, NaN and the largest values; a frequency that is not finite; blocks that are not
    there, tokens of no sequence (their queries are turned all the same), negative starts."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_append_rotary
    heads, dim, block, tokens = 1, 64, 16, 40
    rng = np.random.default_rng(10)
    gpu = KvCache.empty(4, heads, dim, block)
    cache = from_gpu(gpu)
    table = np.array([[2, 0], [1, -1], [3, 4], [-9, 3]], np.int32)  # 4: past the pool
    start = np.array([3, 10, 0, -5], np.int32)
    offsets = np.array([2, 20, 30, 33, 36], np.int32)  # tokens 0, 1 and 36 on belong to nobody
    x = rng.standard_normal((tokens, heads, dim))
    for i, value in enumerate((np.inf, -np.inf, np.nan, 3.3e38, -3.3e38, 1e-40)):
        x[3 + 3 * i, 0, 5 + i] = value
    k = torch.from_numpy(x).to(torch.bfloat16).cuda()
    q = k.expand(tokens, heads, dim).repeat(1, 3, 1)
    positions = rng.integers(0, 99, (2, tokens)).astype(np.int32)
    freq, axis = 1e4 ** (-np.arange(16) / 16), np.arange(16) % 5  # axes past the last are the last
    freq[7] = np.inf
    with np.errstate(all="ignore"):
        got = kv_append_rotary(gpu, q, k, k, int32(table), int32(start), int32(positions),
                               rotary_of(freq, axis, True), offsets=int32(offsets))
        same_queries(got, q, positions, freq, axis, True)
        turned = ko.rotate(plain(k), positions, freq, axis, True).astype(np.float64)
        ko.append(cache, turned, k.double().cpu().numpy(), table[:3], start[:3], offsets[:4])
    same_cache(gpu, cache)


def test_nothing_to_do():
    torch = torch_()
    from hbfsim_b200 import KvCache, KvRotary, kv_append_rotary
    rotary = KvRotary.of(64)
    gpu = KvCache.empty(0, 2, 64)
    none = torch.zeros((2, 0, 2, 64), dtype=torch.float16, device="cuda")
    places = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    assert kv_append_rotary(gpu, none, none, none, table, int32([0, 0]), places, rotary).shape == none.shape
    one = torch.ones((2, 1, 2, 64), dtype=torch.float16, device="cuda")
    got = kv_append_rotary(gpu, one, one, one, table, int32([0, 0]), int32([[0], [1]]), rotary)
    assert torch.equal(got[0], one[0]) and not torch.equal(got[1], one[1])


@pytest.mark.parametrize("bad", ["positions", "axes", "long", "q type", "q heads", "pairs", "gradient", "q gradient",
                                 "freq device"])
def test_refusals(bad):
    torch = torch_()
    from hbfsim_b200 import HbfsimError, KvCache, KvRotary, kv_append_rotary
    gpu = KvCache.empty(2, 1, 64)
    x = torch.ones((1, 1, 1, 64), dtype=torch.float16, device="cuda")
    call = dict(q=x, k=x, v=x, table=int32([[0, 1]]), start=int32([0]), positions=int32([[3]]), rotary=KvRotary.of(64))
    if bad == "positions":
        call["positions"] = int32([[3, 4]])
    elif bad == "axes":
        call["positions"] = int32(np.zeros((5, 1, 1)))
    elif bad == "long":
        call["positions"] = call["positions"].long()
    elif bad == "q type":
        call["q"] = x.to(torch.bfloat16)
    elif bad == "q heads":
        call["q"] = x[0]
    elif bad == "pairs":
        call["rotary"] = KvRotary.of(64, rotated=6)
    elif bad == "gradient":
        call["k"] = x.clone().requires_grad_()
    elif bad == "q gradient":
        call["q"] = x.clone().requires_grad_()
    else:
        with pytest.raises(ValueError):
            KvRotary.of(64, device="cpu")
        return
    with pytest.raises((ValueError, HbfsimError)):
        kv_append_rotary(gpu, **call)
    if "gradient" in bad:
        with torch.no_grad():
            kv_append_rotary(gpu, **call)


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_blocks_begun_and_ended_inside(dim, block):
    """Every number of tokens held before and of new ones that a block can have, in one call; scales
    that grow over what is held and scales that do not; values near the largest of 32 bits."""
    torch = torch_()
    from hbfsim_b200 import KvRotary, kv_append_rotary
    rng = np.random.default_rng(dim + block)
    pairs = [(s, n) for s in range(0, block, 5) for n in (1, 2, 4, 5, 7, 15, 16, 17, 31, 63, 64) if s + n <= block]
    start = np.array([s for s, _ in pairs], np.int32)
    count = np.array([n for _, n in pairs])
    offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    heads, pages, total = 3, len(pairs), int(offsets[-1])
    cache = random_cache(rng, pages, heads, block, dim)
    cache["scale"] *= 2.0 ** rng.integers(-12, 13, cache["scale"].shape)
    cache["scale"][::7] = 2.0 ** 120
    cache["data"][::7] = ko.encode(np.clip(ko.E4M3[cache["data"][::7]], -255, 255))
    cache["data"][3::11, 1, 0, 0, 5] = 0x7f  # held values that are no numbers
    table = rng.permutation(pages).astype(np.int32)[:, None]
    size = 10.0 ** rng.uniform(-4, 4, (total, 1, 1)) * np.where(rng.random((total, 1, 1)) < 0.02, 1e34, 1)
    x = torch.from_numpy(rng.standard_normal((total, 2 * heads, dim)) * size).to(torch.bfloat16).cuda()
    rotary = KvRotary.of(dim, sections=(dim // 4, dim // 4))
    positions = rng.integers(0, 5000, (2, total)).astype(np.int32)
    gpu = to_gpu(cache)
    assert kv_append_rotary(gpu, None, x[:, :heads], x[:, heads:], int32(table), int32(start), int32(positions), rotary,
                            offsets=int32(offsets)) is None
    with np.errstate(over="ignore"):  # some turn into infinities
        turned = ko.rotate(plain(x[:, :heads]), positions, rotary.freq.cpu().numpy(), rotary.axis.cpu().numpy(), False)
    ko.append(cache, turned.astype(np.float64), x[:, heads:].double().cpu().numpy(), table, start, offsets)
    same_cache(gpu, cache)


def test_pool_and_queries_past_32_bit_offsets():
    """Pages behind 2^32 bytes of a pool, tokens behind 2^31 elements of the projection."""
    torch = torch_()
    from hbfsim_b200 import KvCache, KvRotary, kv_append_rotary
    rng = np.random.default_rng(12)
    heads, dim, block = 8, 128, 16
    pages = (1 << 32) // (heads * 2 * block * dim) + 5
    gpu = KvCache.empty(pages, heads, dim, block)
    rotary = KvRotary.of(dim)
    qkv = torch.from_numpy(rng.standard_normal((40, 3 * heads, dim))).to(torch.bfloat16).cuda()
    # 40 tokens whose rows lie 2^26 elements apart: the last 2.6 * 2^30 elements from the first
    far = torch.empty(39 * (1 << 26) + 3 * heads * dim, dtype=torch.bfloat16, device="cuda")
    rows = far.as_strided((40, 3 * heads, dim), (1 << 26, dim, 1))
    rows.copy_(qkv)
    table, start = np.array([[pages - 1, 3, pages - 4]], np.int32), np.array([5], np.int32)
    places = np.arange(40, dtype=np.int32)[None] * 1000
    q, k, v = rows[:, :heads], rows[:, heads:2 * heads], rows[:, 2 * heads:]
    got = kv_append_rotary(gpu, q, k, v, int32(table), int32(start), int32(places), rotary, offsets=int32([0, 40]))
    freq, axis = rotary.freq.cpu().numpy(), rotary.axis.cpu().numpy()
    same_queries(got, qkv[:, :heads], places, freq, axis, False)
    small = KvCache.empty(4, heads, dim, block)
    cache = from_gpu(small)
    turned = ko.rotate(plain(qkv[:, heads:2 * heads]), places, freq, axis, False).astype(np.float64)
    ko.append(cache, turned, qkv[:, 2 * heads:].double().cpu().numpy(), np.array([[0, 1, 2]]), start, [0, 40])
    for there, here in zip(table[0], range(3)):
        assert np.array_equal(ko.E4M3[gpu.data.view(torch.uint8)[int(there)].cpu().numpy()], ko.E4M3[cache["data"][here]])
        assert np.array_equal(gpu.scale[int(there)].double().cpu().numpy(), cache["scale"][here])
        assert np.array_equal(gpu.bounds[int(there)].cpu().numpy(), cache["bounds"][here])
    others = gpu.data.view(torch.uint8).view(pages, -1)
    assert not others[[0, 1, 2, 4, pages - 2, pages - 3, pages - 5]].any()
