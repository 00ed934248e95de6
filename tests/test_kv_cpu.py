"""Refusals of the key/value cache operators: every bad argument is turned
down before any device work (no GPU needed), and the oracle's 8-bit rounding
against the type's own definition."""
import ctypes

import numpy as np
import pytest

import kv_oracle as ko
from hbfsim_b200 import _lib, build

OK, INVALID, UNSUPPORTED = 0, 1, 5


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def cache(**over):
    c = dict(struct_size=ctypes.sizeof(_lib.KvCacheV1), version=1, kv_heads=2, head_dim=128,
             block_tokens=16, reserved=0, pages=4, data=4096, scale=4096, bounds=4096)
    return _lib.KvCacheV1(**{**c, **over})


def append(**over):
    a = dict(struct_size=ctypes.sizeof(_lib.KvAppendBatchV1), version=1, type=0, seqs=2, width=3,
             reserved=0, tokens=4, k=4096, v=4096, k_stride_token=256, k_stride_head=128,
             v_stride_token=256, v_stride_head=128, table=4096, table_stride=3, start=4096,
             offsets=None)
    return _lib.KvAppendBatchV1(**{**a, **over})


def query(**over):
    q = dict(struct_size=ctypes.sizeof(_lib.KvQueryV1), version=1, type=0, seqs=2, tokens=1,
             q_heads=8, width=3, reserved=0, q=4096, q_stride_seq=1024, q_stride_token=1024,
             q_stride_head=128, table=4096, table_stride=3, lengths=4096)
    return _lib.KvQueryV1(**{**q, **over})


def attention(**over):
    a = dict(struct_size=ctypes.sizeof(_lib.KvAttentionArgsV1), version=1, softmax_scale=0.1,
             top=0, blocks=None, counts=None, out=4096, lse=4096, weights=4096, workspace=4096,
             workspace_bytes=1 << 40)
    return _lib.KvAttentionArgsV1(**{**a, **over})


def evict(**over):
    e = dict(struct_size=ctypes.sizeof(_lib.KvEvictBatchV1), version=1, seqs=2, kv_heads=2,
             width=3, block_tokens=16, keep=2, sink=1, recent=1, decay=0, score=4096,
             weights=4096, table=4096, table_stride=3, lengths=4096, score_out=8192,
             table_out=8192, lengths_out=8192, freed=8192, freed_counts=8192)
    return _lib.KvEvictBatchV1(**{**e, **over})


ref = ctypes.byref

CACHES = [(dict(struct_size=1), INVALID), (dict(version=2), INVALID), (dict(reserved=1), INVALID),
          (dict(kv_heads=0), INVALID), (dict(kv_heads=1025), INVALID), (dict(pages=1 << 31), INVALID),
          (dict(head_dim=96), UNSUPPORTED), (dict(block_tokens=24), UNSUPPORTED),
          (dict(data=None), INVALID), (dict(scale=None), INVALID), (dict(bounds=None), INVALID),
          (dict(data=4100), INVALID), (dict(scale=4100), INVALID), (dict(bounds=4100), INVALID)]


@pytest.mark.parametrize("over,rc", CACHES)
def test_cache_refusals(lib, over, rc):
    bad = cache(**over)
    assert lib.hbfsim_kv_append_v1(ref(bad), ref(append()), None) == rc
    assert lib.hbfsim_kv_select_workspace_v1(ref(bad), ref(query())) == 0
    assert lib.hbfsim_kv_select_v1(ref(bad), ref(query()), 2, 1, 1, 4096, 4096, 4096, 1 << 40,
                                   None) == rc
    assert lib.hbfsim_kv_attention_workspace_v1(ref(bad), ref(query()), ref(attention())) == 0
    assert lib.hbfsim_kv_attention_v1(ref(bad), ref(query()), ref(attention()), None) == rc


@pytest.mark.parametrize("over,rc", [
    (dict(struct_size=1), INVALID), (dict(version=0), INVALID), (dict(reserved=1), INVALID),
    (dict(type=2), UNSUPPORTED), (dict(seqs=0), INVALID), (dict(seqs=3), INVALID),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID),
    (dict(start=None), INVALID), (dict(k=4097), INVALID), (dict(offsets=4097), INVALID),
    (dict(tokens=1 << 40), INVALID), (dict(tokens=0, k=None), OK), (dict(width=0), OK)])
def test_append_refusals(lib, over, rc):
    assert lib.hbfsim_kv_append_v1(ref(cache()), ref(append(**over)), None) == rc


QUERIES = [(dict(struct_size=1), INVALID), (dict(version=2), INVALID), (dict(reserved=1), INVALID),
           (dict(type=2), UNSUPPORTED), (dict(tokens=17), UNSUPPORTED), (dict(q_heads=0), INVALID),
           (dict(q_heads=7), INVALID), (dict(q_heads=130), INVALID), (dict(q=None), INVALID),
           (dict(q=4097), INVALID), (dict(table=None), INVALID), (dict(lengths=None), INVALID),
           (dict(lengths=4098), INVALID), (dict(width=1 << 28), INVALID)]


@pytest.mark.parametrize("over,rc", QUERIES + [(dict(seqs=0), OK), (dict(tokens=0), OK)])
def test_query_refusals(lib, over, rc):
    bad = query(**over)
    assert lib.hbfsim_kv_select_v1(ref(cache()), ref(bad), 2, 1, 1, 4096, 4096, 4096, 1 << 40,
                                   None) == rc
    assert lib.hbfsim_kv_attention_v1(ref(cache()), ref(bad), ref(attention()), None) == rc


@pytest.mark.parametrize("top,sink,recent,size,blocks", [
    (0, 0, 0, 1 << 40, 4096), (2, 1, 0, 1 << 40, 4096), (2, 2, 1, 1 << 40, 4096),
    (2, 1, 1, 47, 4096), (2, 1, 1, 1 << 40, None), (2, 1, 1, 1 << 40, 4097)])
def test_select_refusals(lib, top, sink, recent, size, blocks):
    assert lib.hbfsim_kv_select_v1(ref(cache()), ref(query()), top, sink, recent, blocks, 4096, 4096,
                                   size, None) == INVALID


@pytest.mark.parametrize("over", [
    dict(struct_size=1), dict(version=2), dict(softmax_scale=float("nan")),
    dict(softmax_scale=float("inf")), dict(blocks=4096), dict(counts=4096),
    dict(blocks=4096, counts=4096, top=0), dict(out=None), dict(out=4097), dict(lse=4098),
    dict(weights=4098), dict(workspace=None), dict(workspace=4104), dict(workspace_bytes=16)])
def test_attention_refusals(lib, over):
    wide = query(width=5000, table_stride=5000)  # a call that needs a workspace
    assert lib.hbfsim_kv_attention_v1(ref(cache()), ref(wide), ref(attention(**over)),
                                      None) == INVALID


def test_attention_workspace_sizes(lib):
    """Short rows need none; wide ones grow with the sequences and with the weights."""
    size = lambda q, **over: lib.hbfsim_kv_attention_workspace_v1(ref(cache()), ref(q), ref(attention(**over)))
    assert size(query()) == 0
    wide = [size(query(width=5000, seqs=s), weights=w) for s in (2, 4) for w in (None, 4096)]
    assert 0 < wide[0] < wide[1] and wide[0] < wide[2] < wide[3]
    assert all(w % 256 == 0 for w in wide)


def test_packed_structures():
    """The structures that Python packs are those of the header, byte for byte."""
    from hbfsim_b200 import kv
    for packed, struct in ((kv._CACHE, _lib.KvCacheV1), (kv._APPEND, _lib.KvAppendBatchV1),
                           (kv._QUERY, _lib.KvQueryV1), (kv._ATTENTION, _lib.KvAttentionArgsV1),
                           (kv._EVICT, _lib.KvEvictBatchV1)):
        assert packed.size == ctypes.sizeof(struct)
        values = [0.5 if kind is ctypes.c_float else 7 * i + 1
                  for i, (_, kind) in enumerate(struct._fields_)]
        assert packed.pack(*values) == bytes(struct(*values))


@pytest.mark.parametrize("over,rc", [
    (dict(struct_size=1), INVALID), (dict(version=2), INVALID), (dict(block_tokens=8), UNSUPPORTED),
    (dict(kv_heads=0), INVALID), (dict(recent=0), INVALID), (dict(keep=1), INVALID),
    (dict(sink=2), INVALID), (dict(decay=64), INVALID), (dict(score=None), INVALID),
    (dict(weights=None), INVALID), (dict(table=None), INVALID), (dict(lengths=None), INVALID),
    (dict(score_out=4096), INVALID), (dict(table_out=4096), INVALID), (dict(freed=None), INVALID),
    (dict(freed_counts=None), INVALID), (dict(lengths_out=None), INVALID),
    (dict(score=4100), INVALID), (dict(width=1 << 28), INVALID), (dict(seqs=0), OK)])
def test_evict_refusals(lib, over, rc):
    assert lib.hbfsim_kv_evict_v1(ref(evict(**over)), None) == rc


def test_null_structures(lib):
    assert lib.hbfsim_kv_append_v1(None, None, None) == INVALID
    assert lib.hbfsim_kv_append_v1(ref(cache()), None, None) == INVALID
    assert lib.hbfsim_kv_attention_v1(ref(cache()), ref(query()), None, None) == INVALID
    assert lib.hbfsim_kv_attention_v1(ref(cache()), None, ref(attention()), None) == INVALID
    assert lib.hbfsim_kv_evict_v1(None, None) == INVALID


def test_python_refusals():
    """Shapes and types that do not fit raise before the library is called."""
    torch = pytest.importorskip("torch")
    from hbfsim_b200 import KvCache, kv_evict
    data = torch.zeros((2, 1, 2, 16, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale, bounds = torch.ones((2, 1, 2)), torch.zeros((2, 1, 2, 64), dtype=torch.int8)
    for bad in ((data.view(torch.uint8), scale, bounds), (data, scale.double(), bounds),
                (data, scale[:1], bounds), (data, scale, bounds[..., :32]),
                (data, scale, bounds)):  # the last: not on a CUDA device
        with pytest.raises(ValueError):
            KvCache(*bad)
    with pytest.raises(ValueError):
        kv_evict(torch.zeros((1, 3), dtype=torch.int64), torch.zeros((1, 1, 3)),
                 torch.zeros((1, 3), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), keep=2)


def test_oracle_rounding_matches_the_type():
    """oracle encode() against torch's float8_e4m3fn cast inside its range: every value, every
    midpoint, their neighbours, and random values."""
    torch = pytest.importorskip("torch")
    grid = ko._MAGNITUDES
    mid = (grid[1:] + grid[:-1]) / 2
    rng = np.random.default_rng(0)
    x = np.concatenate([grid, mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                        np.nextafter(mid.astype(np.float32), np.float32(1e9)),
                        448 * rng.random(2000), 2.0 ** rng.uniform(-12, 8, 2000)])
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ko.E4M3[ko.encode(x)], ko.E4M3[want])
    assert ko.encode(np.array([1e9, -np.inf])).tolist() == [126, 254]
    assert ko.encode(np.array([np.nan])).tolist() == [127]


# kv_evict with every array where it has room of its own: 2 sequences of 3 blocks, 2 heads
APART = dict(score=0x10000, weights=0x20000, table=0x30000, lengths=0x40000, score_out=0x50000,
             table_out=0x60000, lengths_out=0x70000, freed=0x80000, freed_counts=0x90000)


@pytest.mark.parametrize("over", [
    dict(lengths=0x40002), dict(lengths_out=0x70002), dict(freed_counts=0x90002),  # not of 4 bytes
    # an output in an input's memory
    dict(lengths_out=0x40000), dict(lengths_out=0x40004), dict(freed_counts=0x40000),
    dict(freed=0x30000), dict(table_out=0x30014), dict(score_out=0x10028), dict(score_out=0x0ffd8),
    dict(table_out=0x20000), dict(freed=0x2002c), dict(score_out=0x30008), dict(table_out=0x10000),
    dict(lengths_out=0x10000), dict(freed_counts=0x30000),
    dict(table_stride=100, freed=0x30000 + 400), dict(table_stride=-3, freed=0x30000 - 12),
    # outputs in each other's
    dict(lengths_out=0x90004), dict(freed=0x60000), dict(table_out=0x80014), dict(freed=0x50000 + 44)])
def test_evict_refuses_memory_that_would_race(lib, over):
    assert lib.hbfsim_kv_evict_v1(ref(evict(**{**APART, **over})), None) == INVALID
