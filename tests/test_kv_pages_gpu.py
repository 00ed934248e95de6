"""kv_resize, kv_fork, kv_copy and kv_compact against their definitions (oracle/kv_oracle.py):
equal, by one cluster of thread blocks and by a launch to a pass (pools of more than 2^19 counts and
entries)."""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import from_gpu, int32, random_cache, to_gpu, torch_

pytestmark = pytest.mark.gpu

LARGE = 700000  # pages past the cluster's form


def counted(table, pages):
    real = table[(table >= 0) & (table < pages)]
    return np.bincount(real.ravel(), minlength=pages).astype(np.int32)


def pool(rng, seqs, width, pages, block, share=0.3, holes=0.02, fill=0.7):
    """A table whose rows share some of their first pages, with holes and entries past the pool;
    counts that fit it, a few pages held by no table."""
    lengths = rng.integers(0, width * block + 1, seqs).astype(np.int32)
    lengths = np.minimum(lengths, rng.integers(0, int(fill * width * block) + 2, seqs)).astype(np.int32)
    table = np.full((seqs, width), -1, np.int32)
    order = rng.permutation(pages).tolist()
    for b in range(seqs):
        have = -(-int(lengths[b]) // block)
        row = [order.pop() if order else -1 for _ in range(have)]
        if b and rng.random() < share and have:
            other = table[rng.integers(0, b)]
            many = min(have, int((other >= 0).sum()), int(rng.integers(1, have + 1)))
            row[:many] = other[:many]
        table[b, :have] = row
        if have and rng.random() < holes * have:
            table[b, rng.integers(0, have)] = rng.choice([-1, pages, -9])
    refs = counted(table, pages)
    for p in order[:3]:
        refs[p] += 1
    return refs, table, lengths


def same(got, want):
    for g, w, name in zip(got, want, got._fields):
        assert np.array_equal(g.cpu().numpy(), w), name


def resize_and_check(refs, table, lengths, want, block=16, freed=None, freed_counts=None, stream=None):
    from hbfsim_b200 import kv_resize
    expected = ko.resize(refs, table, lengths, want, block, freed, freed_counts)
    listed = {} if freed is None else dict(freed=int32(freed), freed_counts=int32(freed_counts))
    r, t = int32(refs), int32(table)
    got = kv_resize(r, t, int32(lengths), int32(want), block, stream=stream, **listed)
    same(got, expected)
    assert np.array_equal(r.cpu().numpy(), refs) and np.array_equal(t.cpu().numpy(), table), "inputs"
    # in place, in rows of a wider tensor
    wide = int32(np.pad(table, ((0, 0), (0, 3)), constant_values=77))
    view = wide[:, :table.shape[1]]
    got = kv_resize(r, view, int32(lengths), int32(want), block, inplace=True, stream=stream, **listed)
    assert got.refs is r and got.table is view
    same(got, expected)
    assert (wide[:, table.shape[1]:] == 77).all()
    return expected


RESIZES = [  # seqs, width, pages, block
    (1, 1, 1, 16), (1, 3, 4, 16), (5, 4, 30, 16), (64, 40, 3000, 16), (64, 40, 900, 16), (33, 17, 500, 32),
    (8, 600, 5000, 64), (300, 5, 1100, 16), (3, 3000, 20000, 16), (1200, 3, 5000, 16), (2, 40, LARGE, 16),
    (900, 600, 300000, 16)]


@pytest.mark.parametrize("seqs,width,pages,block", RESIZES)
def test_resize(seqs, width, pages, block):
    """Rows that end, shrink, stay, take a token and take a prompt; pools that run out."""
    rng = np.random.default_rng(seqs + width + pages)
    refs, table, lengths = pool(rng, seqs, width, pages, block)
    kind = rng.integers(0, 6, seqs)
    want = np.select([kind == 0, kind == 1, kind == 2, kind == 3, kind == 4],
                     [0 * lengths, lengths // 2, lengths, lengths + 1, lengths + rng.integers(0, 5 * block, seqs)],
                     rng.integers(-5, width * block + 9, seqs)).astype(np.int32)
    freed = rng.integers(-2, pages + 2, (seqs, 4)).astype(np.int32)
    counts = rng.integers(-1, 6, seqs).astype(np.int32)
    refs += counted(np.where(np.arange(4) < counts[:, None], freed, -1), pages)
    out = resize_and_check(refs, table, lengths, want, block, freed, counts)
    # a step further, from where it ended
    resize_and_check(out[0], out[1], out[2], out[2] + 1, block)


@pytest.mark.parametrize("sharers,free", [(2, 0), (2, 1), (4, 2), (4, 3), (5, 9), (40, 38), (40, 100)])
def test_shared_last_blocks_are_parted(sharers, free):
    """The last one that asks for a page keeps it, if all others got theirs; one that does not ask
    keeps its share."""
    for extra in (0, 1):  # one sharer more, which does not grow
        seqs, width, block = sharers + extra, 2, 16
        pages = 1 + free
        table = np.full((seqs, width), -1, np.int32)
        table[:, 0] = pages - 1
        lengths = np.full(seqs, 5, np.int32)
        want = lengths + 1
        if extra:
            want[seqs // 2] = 5
        refs = counted(table, pages)
        out = resize_and_check(refs, table, lengths, want, block)
        parted = (out[3] >= 0).sum()
        assert parted == min(free, sharers - 1 + extra)


@pytest.mark.parametrize("seqs,width,rows,pages,block", [
    (1, 1, 1, 1, 16), (4, 3, 9, 20, 16), (64, 40, 64, 3000, 16), (7, 100, 300, 2000, 32), (30, 9, 4, 300, 64),
    (5, 4, 0, 50, 16), (2, 0, 3, 10, 16), (3, 40, 5, LARGE, 16), (900, 600, 40, 300000, 16), (10, 500, 1300, 4000, 16)])
def test_fork(seqs, width, rows, pages, block):
    torch = torch_()
    from hbfsim_b200 import kv_fork
    rng = np.random.default_rng(seqs + rows)
    refs, table, lengths = pool(rng, seqs, width, pages, block, fill=1.2)
    if width:
        table[rng.random(table.shape) < 0.01] = 0  # named behind a row's end too
    refs = counted(table, pages)
    parents = rng.integers(-2, seqs + 2, rows).astype(np.int32)
    parents[:rows // 2] = np.arange(rows // 2)  # half go on as themselves
    want = ko.fork(refs, table, lengths, parents, block)
    for inplace in (False, True):
        r = int32(refs)
        got = kv_fork(r, int32(table), int32(lengths), int32(parents), block, inplace=inplace)
        same(got, want)
        assert (got.refs is r) == inplace and (inplace or np.array_equal(r.cpu().numpy(), refs))
        assert torch.equal(got.refs, int32(counted(want[1], pages)))


@pytest.mark.parametrize("pages,seqs,width,live", [
    (1, 1, 1, 1.0), (2, 1, 2, 0.5), (7, 2, 3, 0.0), (50, 4, 5, 0.4), (1024, 9, 33, 0.5), (1025, 3, 600, 0.9),
    (20000, 60, 70, 0.02), (60000, 5, 9, 0.99), (LARGE, 3, 50, 0.5), (30000, 900, 600, 0.3), (0, 2, 3, 0.0)])
def test_compact(pages, seqs, width, live):
    from hbfsim_b200 import kv_compact
    rng = np.random.default_rng(pages + seqs)
    refs = np.where(rng.random(pages) < live, rng.integers(1, 5, pages), rng.integers(-2, 1, pages)).astype(np.int32)
    table = rng.integers(-3, pages + 3, (seqs, width)).astype(np.int32)
    want = ko.compact(refs, table)
    r, t = int32(refs), int32(table)
    same(kv_compact(r, t), want)
    assert np.array_equal(r.cpu().numpy(), refs) and np.array_equal(t.cpu().numpy(), table)
    wide = int32(np.pad(table, ((0, 0), (2, 1))))
    got = kv_compact(r, wide[:, 2:-1], inplace=True)
    same(got, want)
    assert got.refs is r and not wide[:, :2].any() and not wide[:, -1].any()


@pytest.mark.parametrize("dim,block,heads,pages", [(64, 16, 1, 9), (128, 16, 8, 40), (256, 64, 3, 12), (64, 32, 5, 300)])
def test_copy(dim, block, heads, pages):
    """Pages inside one cache and from another; entries outside either pool are passed over."""
    from hbfsim_b200 import kv_copy
    rng = np.random.default_rng(dim + pages)
    cache, other = random_cache(rng, pages, heads, block, dim), random_cache(rng, 5, heads, block, dim)
    order = rng.permutation(pages)
    many = pages // 2
    src, dst = order[:many].copy(), order[many:2 * many].copy()
    src[0], dst[1] = -1, pages
    gpu = to_gpu(cache)
    kv_copy(gpu, int32(src), int32(dst))
    for a, b in zip(src[2:], dst[2:]):
        for x in cache.values():
            x[b] = x[a]
    compare = from_gpu(gpu)
    for name, x in cache.items():
        assert np.array_equal(compare[name], x), name
    kv_copy(gpu, int32([4, 5, 0, -1]), int32([0, 1, 2, 3]), source=to_gpu(other))
    for x, y in zip(cache.values(), other.values()):
        x[0], x[2] = y[4], y[0]
    compare = from_gpu(gpu)
    for name, x in cache.items():
        assert np.array_equal(compare[name], x), name
    kv_copy(gpu, int32([]), int32([]))


def test_copy_past_32_bit_offsets():
    """A pool of more than 2^32 bytes: from its end to its beginning and back."""
    torch = torch_()
    from hbfsim_b200 import KvCache, kv_copy
    pages = (1 << 32) // 32768 + 10
    gpu = KvCache.empty(pages, 8, 128, 16)
    data = gpu.data.view(torch.uint8)
    data[pages - 3] = 7
    gpu.scale[pages - 3] = 4.0
    gpu.bounds[pages - 3] = -5
    data[4] = 9
    kv_copy(gpu, int32([pages - 3, 4]), int32([1, pages - 1]))
    assert (data[1] == 7).all() and (gpu.scale[1] == 4).all() and (gpu.bounds[1] == -5).all()
    assert (data[pages - 1] == 9).all() and not data[0].any() and not data[2].any() and not data[pages - 2].any()


@pytest.mark.parametrize("bad", ["refs", "refs long", "want", "block", "freed", "freed counts", "parents", "src",
                                 "shapes", "cpu", "overlap"])
def test_refusals(bad):
    torch = torch_()
    from hbfsim_b200 import HbfsimError, KvCache, kv_compact, kv_copy, kv_fork, kv_resize
    refs, table, one = int32(np.ones(8)), int32(np.arange(8).reshape(2, 4)), int32([16, 16])
    with pytest.raises((ValueError, HbfsimError)):
        if bad == "refs":
            kv_compact(refs.view(2, 4), table)
        elif bad == "refs long":
            kv_compact(refs.long(), table)
        elif bad == "want":
            kv_resize(refs, table, one, int32([3]))
        elif bad == "block":
            kv_resize(refs, table, one, one, block_tokens=24)
        elif bad == "freed":
            kv_resize(refs, table, one, one, freed=table)
        elif bad == "freed counts":
            kv_resize(refs, table, one, one, freed_counts=one)
        elif bad == "parents":
            kv_fork(refs, table, one, int32([[0]]))
        elif bad == "src":
            kv_copy(KvCache.empty(2, 1, 64), int32([0]), int32([0, 1]))
        elif bad == "shapes":
            kv_copy(KvCache.empty(2, 1, 64), int32([0]), int32([1]), source=KvCache.empty(2, 1, 128))
        elif bad == "cpu":
            kv_resize(refs.cpu(), table, one, one)
        else:  # rows of the table in one another cannot be changed in place
            kv_resize(refs, table.flatten().as_strided((2, 4), (2, 1)), one, one, inplace=True)


@pytest.mark.parametrize("seqs,width,pages", [(0, 3, 5), (0, 0, 0), (3, 0, 5), (3, 4, 0), (1, 1, 0)])
def test_nothing_there(seqs, width, pages):
    """No sequences, no room in the table, no pages."""
    from hbfsim_b200 import KvCache, kv_compact, kv_copy, kv_fork
    refs, table = np.zeros(pages, np.int32), np.full((seqs, width), -1, np.int32)
    lengths = np.zeros(seqs, np.int32)
    freed = np.full((2, 3), 1, np.int32)
    out = resize_and_check(refs, table, lengths, lengths + 20, 16, freed, np.array([2, 3]))
    assert (out[2] == 0).all() or width == 0 or pages
    parents = np.array([0, -1, 5], np.int32)
    same(kv_fork(int32(refs), int32(table), int32(lengths), int32(parents)), ko.fork(refs, table, lengths, parents, 16))
    same(kv_compact(int32(refs), int32(table)), ko.compact(refs, table))
    if pages == 0:
        kv_copy(KvCache.empty(0, 1, 64), int32([0, -1, 3]), int32([0, 1, 2]))


def test_rows_that_are_one_row():
    """A table whose rows are one row in memory (as expand gives it): every row counts."""
    from hbfsim_b200 import kv_fork, kv_resize
    row = int32([[2, 0, -1]])
    refs = np.array([4, 0, 4, 0], np.int32)
    table, lengths = row.expand(4, 3), np.array([20, 20, 20, 20], np.int32)
    plain = row.cpu().numpy().repeat(4, 0)
    same(kv_resize(int32(refs), table, int32(lengths), int32(lengths - 10)), ko.resize(refs, plain, lengths, lengths - 10, 16))
    same(kv_fork(int32(refs), table, int32(lengths), int32([1, 1])), ko.fork(refs, plain, lengths, [1, 1], 16))
