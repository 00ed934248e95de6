"""Refusals of the operators around the attention (positions, drafted tokens, pages): every bad
argument is turned down before any device work (no GPU needed); and their oracle against what
follows from the definitions."""
import ctypes

import numpy as np
import pytest

import kv_oracle as ko
from hbfsim_b200 import _lib, build
from test_kv_cpu import CACHES, INVALID, OK, UNSUPPORTED, append, cache

ref = ctypes.byref


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def make(struct, defaults, over):
    return struct(struct_size=ctypes.sizeof(struct), version=1, **{**defaults, **over}) \
        if not {"struct_size", "version"} & set(over) else \
        struct(**{**dict(struct_size=ctypes.sizeof(struct), version=1), **defaults, **over})


def rotary(**over):
    return make(_lib.KvRotaryV1, dict(
        q_heads=8, axes=3, pairs=64, neighbours=0, q=4096, q_stride_token=1024, q_stride_head=128,
        q_out=4096, positions=4096, positions_stride=4, freq=4096, axis=4096), over)


def verify(**over):
    return make(_lib.KvVerifyBatchV1, dict(
        type=2, seqs=2, drafts=3, vocab=100, target=4096, target_stride_seq=400,
        target_stride_token=100, draft=4096, draft_stride_seq=300, draft_stride_token=100,
        tokens=4096, accept=4096, sample=4096, counts=4096, lengths=4096, accepted=8192,
        tokens_out=8192, lengths_out=8192), over)


# 4 sequences of 6 blocks, 100 pages, every array with room of its own
def resize(**over):
    return make(_lib.KvResizeBatchV1, dict(
        seqs=4, width=6, block_tokens=16, freed_rows=4, freed_width=6, reserved=0, pages=100,
        refs=0x10000, table=0x20000, table_stride=6, lengths=0x30000, want=0x40000, freed=0x50000,
        freed_counts=0x60000, refs_out=0x70000, table_out=0x80000, table_out_stride=6,
        limits=0x90000, src=0xa0000, dst=0xb0000, workspace=0x100000, workspace_bytes=1 << 20), over)


def fork(**over):
    return make(_lib.KvForkBatchV1, dict(
        seqs=4, rows=5, width=6, block_tokens=16, pages=100, refs=0x10000, table=0x20000,
        table_stride=6, lengths=0x30000, parents=0x40000, refs_out=0x70000, table_out=0x80000,
        lengths_out=0x90000), over)


def compact(**over):
    return make(_lib.KvCompactBatchV1, dict(
        seqs=4, width=6, pages=100, refs=0x10000, table=0x20000, table_stride=6, refs_out=0x70000,
        table_out=0x80000, table_out_stride=6, src=0x90000, dst=0xa0000, live=0xb0000,
        where=0xc0000, workspace=0x100000, workspace_bytes=1 << 20), over)


@pytest.mark.parametrize("over,rc", CACHES)
def test_cache_refusals(lib, over, rc):
    bad = cache(**over)
    assert lib.hbfsim_kv_append_rotary_v1(ref(bad), ref(append()), ref(rotary()), None) == rc
    assert lib.hbfsim_kv_copy_v1(ref(bad), ref(cache()), 4096, 4096, 3, None) == rc
    assert lib.hbfsim_kv_copy_v1(ref(cache()), ref(bad), 4096, 4096, 3, None) == rc


@pytest.mark.parametrize("over,rc", [
    (dict(struct_size=1), INVALID), (dict(version=0), INVALID), (dict(reserved=1), INVALID),
    (dict(type=2), UNSUPPORTED), (dict(seqs=3), INVALID), (dict(k=None), INVALID),
    (dict(start=None), INVALID), (dict(tokens=1 << 40), INVALID), (dict(tokens=0, k=None), OK)])
def test_rotary_refuses_a_bad_append(lib, over, rc):
    assert lib.hbfsim_kv_append_rotary_v1(ref(cache()), ref(append(**over)), ref(rotary()), None) == rc


@pytest.mark.parametrize("over,rc", [
    (dict(struct_size=1), INVALID), (dict(version=2), INVALID), (dict(axes=0), INVALID),
    (dict(axes=5), INVALID), (dict(neighbours=2), INVALID), (dict(q_heads=65537), INVALID),
    (dict(pairs=0), UNSUPPORTED), (dict(pairs=65), UNSUPPORTED), (dict(pairs=68), UNSUPPORTED),
    (dict(pairs=6), UNSUPPORTED), (dict(q=None), INVALID), (dict(q=4097), INVALID),
    (dict(q_out=None), INVALID), (dict(q_out=4104), INVALID), (dict(positions=None), INVALID),
    (dict(positions=4098), INVALID), (dict(freq=None), INVALID), (dict(freq=4100), INVALID),
    (dict(axis=None), INVALID)])
def test_rotary_refusals(lib, over, rc):
    assert lib.hbfsim_kv_append_rotary_v1(ref(cache()), ref(append()), ref(rotary(**over)), None) == rc


def test_rotary_without_queries_and_blocks_does_nothing(lib):
    call = lib.hbfsim_kv_append_rotary_v1
    assert call(ref(cache()), ref(append(width=0)), ref(rotary(q_heads=0, q=None, q_out=None)), None) == OK


@pytest.mark.parametrize("over,rc", [
    (dict(struct_size=1), INVALID), (dict(version=2), INVALID), (dict(type=3), UNSUPPORTED),
    (dict(drafts=33), UNSUPPORTED), (dict(vocab=0), INVALID), (dict(vocab=(1 << 22) + 1), INVALID),
    (dict(seqs=65537), INVALID), (dict(target=None), INVALID), (dict(target=4098), INVALID),
    (dict(draft=4098), INVALID), (dict(tokens=None), INVALID), (dict(accept=None), INVALID),
    (dict(sample=None), INVALID), (dict(accepted=None), INVALID), (dict(tokens_out=None), INVALID),
    (dict(lengths=None), INVALID), (dict(counts=4097), INVALID), (dict(sample=4097), INVALID),
    (dict(tokens_out=4098), INVALID), (dict(seqs=0), OK)])
def test_verify_refusals(lib, over, rc):
    assert lib.hbfsim_kv_verify_v1(ref(verify(**over)), None) == rc


TABLES = [  # for every operator on pages
    (dict(struct_size=1), INVALID), (dict(version=2), INVALID), (dict(seqs=65537), INVALID),
    (dict(width=(1 << 24) + 1), INVALID), (dict(seqs=65536, width=1 << 15), INVALID),
    (dict(pages=1 << 31), INVALID), (dict(refs=None), INVALID), (dict(refs=0x10002), INVALID),
    (dict(table=None), INVALID), (dict(table=0x20002), INVALID), (dict(refs_out=None), INVALID),
    (dict(table_out=None), INVALID), (dict(refs_out=0x10004), INVALID),
    (dict(refs_out=0x20000), INVALID), (dict(table_out=0x20004), INVALID),
    (dict(table_out=0x10000), INVALID), (dict(refs_out=0x80000 - 4), INVALID)]


@pytest.mark.parametrize("over,rc", TABLES + [
    (dict(reserved=1), INVALID), (dict(block_tokens=8), UNSUPPORTED), (dict(lengths=None), INVALID),
    (dict(want=None), INVALID), (dict(want=0x40001), INVALID), (dict(limits=None), INVALID),
    (dict(src=None), INVALID), (dict(dst=None), INVALID), (dict(freed=None), INVALID),
    (dict(freed_counts=None), INVALID), (dict(freed_rows=1 << 31, freed_width=2), INVALID),
    (dict(workspace=None), INVALID), (dict(workspace=0x100008), INVALID),
    (dict(workspace_bytes=1000), INVALID), (dict(workspace=0x70000), INVALID),
    (dict(limits=0xa0000), INVALID), (dict(src=0xb0008), INVALID), (dict(dst=0x30000), INVALID),
    (dict(limits=0x40000), INVALID), (dict(src=0x60000), INVALID), (dict(dst=0x50010), INVALID),
    # in place: with the table's own rows
    (dict(table_out=0x20000, table_out_stride=8), INVALID), (dict(table_out_stride=5), INVALID),
    (dict(table_out_stride=0), INVALID),
    (dict(seqs=0, freed_rows=0, refs_out=0x10000), OK)])
def test_resize_refusals(lib, over, rc):
    assert lib.hbfsim_kv_resize_v1(ref(resize(**over)), None) == rc


@pytest.mark.parametrize("over,rc", TABLES + [
    (dict(block_tokens=24), UNSUPPORTED), (dict(rows=65537), INVALID), (dict(lengths=None), INVALID),
    (dict(parents=None), INVALID), (dict(lengths_out=None), INVALID), (dict(parents=0x40002), INVALID),
    (dict(table_out=0x20000), INVALID), (dict(lengths_out=0x30000), INVALID),
    (dict(lengths_out=0x80010), INVALID), (dict(seqs=0, rows=0, refs_out=0x10000), OK)])
def test_fork_refusals(lib, over, rc):
    assert lib.hbfsim_kv_fork_v1(ref(fork(**over)), None) == rc


@pytest.mark.parametrize("over,rc", TABLES + [
    (dict(src=None), INVALID), (dict(dst=None), INVALID), (dict(live=None), INVALID),
    (dict(where=None), INVALID), (dict(where=0x10000), INVALID), (dict(live=0x90010), INVALID),
    (dict(src=0xa0004), INVALID), (dict(workspace=None), INVALID),
    (dict(workspace_bytes=64), INVALID), (dict(table_out=0x20000, table_out_stride=7), INVALID)])
def test_compact_refusals(lib, over, rc):
    assert lib.hbfsim_kv_compact_v1(ref(compact(**over)), None) == rc


@pytest.mark.parametrize("over,src,dst,count,rc", [
    (dict(kv_heads=3), 4096, 4096, 3, INVALID), (dict(head_dim=64), 4096, 4096, 3, INVALID),
    (dict(block_tokens=32), 4096, 4096, 3, INVALID), ({}, None, 4096, 3, INVALID),
    ({}, 4096, None, 3, INVALID), ({}, 4098, 4096, 3, INVALID), ({}, 4096, 4096, 1 << 31, INVALID),
    ({}, None, None, 0, OK)])
def test_copy_refusals(lib, over, src, dst, count, rc):
    assert lib.hbfsim_kv_copy_v1(ref(cache(**over)), ref(cache()), src, dst, count, None) == rc


def test_workspace_sizes(lib):
    size = lambda **over: lib.hbfsim_kv_resize_workspace_v1(ref(resize(**over)))  # noqa: E731
    assert 0 < size() < size(pages=10000) and size(width=6000) > size()
    assert size(block_tokens=8) == 0 and lib.hbfsim_kv_resize_workspace_v1(None) == 0
    assert lib.hbfsim_kv_compact_workspace_v1(ref(compact())) > 0
    assert lib.hbfsim_kv_compact_workspace_v1(ref(compact(version=3))) == 0


def test_null_structures(lib):
    assert lib.hbfsim_kv_append_rotary_v1(ref(cache()), ref(append()), None, None) == INVALID
    assert lib.hbfsim_kv_append_rotary_v1(None, ref(append()), ref(rotary()), None) == INVALID
    for name in ("verify", "resize", "fork", "compact"):
        assert getattr(lib, f"hbfsim_kv_{name}_v1")(None, None) == INVALID
    assert lib.hbfsim_kv_copy_v1(None, ref(cache()), 4096, 4096, 1, None) == INVALID


def test_packed_structures():
    """The structures that Python packs are those of the header, byte for byte."""
    from hbfsim_b200 import kv
    for packed, struct in (((kv._ROTARY,), _lib.KvRotaryV1), ((kv._VERIFY,), _lib.KvVerifyBatchV1),
                           ((kv._RESIZE, kv._WORKSPACE), _lib.KvResizeBatchV1),
                           ((kv._FORK,), _lib.KvForkBatchV1),
                           ((kv._COMPACT, kv._WORKSPACE), _lib.KvCompactBatchV1)):
        assert sum(p.size for p in packed) == ctypes.sizeof(struct)
        values = [7 * i + 1 for i in range(len(struct._fields_))]
        rest = 2 if len(packed) == 2 else 0
        parts = (values[:len(values) - rest], values[len(values) - rest:])
        assert b"".join(p.pack(*v) for p, v in zip(packed, parts)) == bytes(struct(*values))


def test_python_refusals():
    """Tensors that are not on a CUDA device raise before the library is called."""
    torch = pytest.importorskip("torch")
    from hbfsim_b200 import KvRotary, kv_compact, kv_fork, kv_resize, kv_verify
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        kv_verify(torch.zeros((1, 3, 8)), None, i32(1, 2), torch.zeros((1, 2)), torch.zeros(1))
    for call in (lambda: kv_resize(i32(4), i32(1, 3), i32(1), i32(1)),
                 lambda: kv_fork(i32(4), i32(1, 3), i32(1), i32(1)),
                 lambda: kv_compact(i32(4), i32(1, 3)),
                 lambda: KvRotary(torch.zeros(64, dtype=torch.float64), torch.zeros(64, dtype=torch.uint8)),
                 lambda: KvRotary(torch.zeros(64), torch.zeros(64, dtype=torch.uint8)),
                 lambda: KvRotary.of(128, rotated=130, device="cpu"),
                 lambda: KvRotary.of(128, rotated=63, device="cpu"),
                 lambda: KvRotary.of(128, sections=(16, 24), device="cpu"),
                 lambda: KvRotary.of(128, sections=(64, 0, 0, 0, 0), device="cpu")):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------------------
# the oracle


@pytest.mark.parametrize("neighbours", [False, True])
def test_oracle_turns_keep_lengths_and_relative_positions(neighbours):
    """A turn keeps every pair's length, and the product of two turned vectors depends on the
    distance of their positions alone."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 1, 64))
    freq, axis = 100.0 ** (-np.arange(32) / 32), np.zeros(32, int)
    at = lambda a, b: ko.rotate(x, np.array([[a, b]]), freq, axis, neighbours).astype(np.float64)  # noqa: E731
    near, far = at(5, 12), at(100005, 100012)
    assert np.allclose(np.linalg.norm(near, axis=-1), np.linalg.norm(x, axis=-1), rtol=1e-5)
    assert abs((near[0, 0] @ near[1, 0]) - (far[0, 0] @ far[1, 0])) < 64 * 2.0 ** -22
    assert not np.allclose(near, far, atol=0.1)
    assert np.array_equal(at(0, 0), x.astype(np.float32))


def test_oracle_verify_draws_from_the_target():
    """Tokens drawn from the draft and verified come out with the target's distribution: over all
    (draft token, accept, sample) on a grid, each token as often as the target says."""
    target = np.array([[[0.5, 0.25, 0.125, 0.125], [0.25] * 4]], np.float32)
    draft = np.array([[[0.125, 0.5, 0.25, 0.125]]], np.float32)
    mass = np.zeros(4)
    grid = (np.arange(8) + 0.5) / 8
    for t in range(4):
        for u in grid:
            for s in grid:
                _, out, _ = ko.verify(target, draft, np.array([[t]]), np.array([[u]]), np.array([s]), [1], [9])
                mass[out[0, 0]] += draft[0, 0, t] / 64
    assert np.allclose(mass, target[0, 0], atol=1 / 64)


def test_oracle_pages_stay_counted():
    """Random resizes, forks and compactions: counts are always what the table says."""
    rng = np.random.default_rng(5)
    pages, width, block = 40, 6, 16
    table, lengths = np.full((5, width), -1, np.int32), np.zeros(5, np.int32)
    refs = np.zeros(pages, np.int32)
    counted = lambda t: np.bincount(t[t >= 0].ravel(), minlength=pages)  # noqa: E731
    for step in range(60):
        want = np.where(rng.random(5) < 0.2, 0, lengths + rng.integers(0, 30, 5)).astype(np.int32)
        refs, table, limits, src, dst = ko.resize(refs, table, lengths, want, block)
        assert (limits <= want).all() and (limits >= np.minimum(lengths, want)).all()
        assert np.array_equal(refs, counted(table))
        # what a sequence may be filled up to lies in pages of its own
        for b in range(5):
            for j in range(lengths[b] // block, -(-int(limits[b]) // block)):
                if limits[b] > lengths[b]:
                    assert refs[table[b, j]] == 1
        lengths = limits
        if step % 3 == 0:
            refs, table, lengths = ko.fork(refs, table, lengths, rng.integers(-1, 5, 5), block)
            assert np.array_equal(refs, counted(table))
        if step % 7 == 0:
            refs, table, _, _, live, _ = ko.compact(refs, table)
            assert np.array_equal(refs, counted(table)) and (refs[:live[0]] > 0).all()
