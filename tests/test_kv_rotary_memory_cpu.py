"""kv_append_rotary turns down queries that would be written into the inputs' or the cache's memory,
before any device work (no GPU needed)."""
import ctypes

import pytest

from hbfsim_b200 import _lib, build
from test_kv_cpu import INVALID, OK

ref = ctypes.byref
# 2 sequences of 4 tokens, 2 key/value heads and 4 query heads of 64 channels, 10 pages of 16 tokens;
# every array 1 MB from the next
CACHE = dict(kv_heads=2, head_dim=64, block_tokens=16, pages=10, data=0x100000, scale=0x200000, bounds=0x300000)
APPEND = dict(type=0, seqs=2, width=3, tokens=8, k=0x400000, v=0x500000, k_stride_token=128, k_stride_head=64,
              v_stride_token=128, v_stride_head=64, table=0x600000, table_stride=3, start=0x700000, offsets=0x800000)
ROTARY = dict(q_heads=4, axes=3, pairs=32, q=0x900000, q_stride_token=256, q_stride_head=64, q_out=0xa00000,
              positions=0xb00000, positions_stride=8, freq=0xc00000, axis=0xd00000)
OUT = 8 * 4 * 64 * 2  # bytes of the turned queries


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def call(lib, append={}, rotary={}):
    of = lambda struct, *given: struct(  # noqa: E731
        struct_size=ctypes.sizeof(struct), version=1, **{k: v for g in given for k, v in g.items()})
    return lib.hbfsim_kv_append_rotary_v1(ref(of(_lib.KvCacheV1, CACHE)), ref(of(_lib.KvAppendBatchV1, APPEND, append)),
                                          ref(of(_lib.KvRotaryV1, ROTARY, rotary)), None)


@pytest.mark.parametrize("at", [
    0x100000, 0x100000 + 10 * 2 * 2 * 16 * 64 - 16, 0x200000 + 10 * 2 * 2 * 4 - 16, 0x300000, 0x300000 + 10 * 2 * 2 * 64 - 16,
    0x400000 - OUT + 16, 0x400000 + 8 * 2 * 64 * 2 - 16, 0x500000, 0x500000 + 8 * 2 * 64 * 2 - 16, 0x600000 + 16, 0x700000,
    0x800000, 0x900000, 0x900000 + 16, 0x900000 + OUT - 16, 0xb00000 + 3 * 8 * 4 - 16, 0xc00000 + 32 * 8 - 16,
    0xd00000 + 16])
def test_turned_queries_in_other_memory_are_refused(lib, at):
    assert call(lib, rotary=dict(q_out=at)) == INVALID


def test_rows_between_which_the_queries_would_lie(lib):
    assert call(lib, append=dict(k_stride_token=1 << 20), rotary=dict(q_out=0x400000 + (1 << 20))) == INVALID
    assert call(lib, rotary=dict(q=0xa00000 + 7 * 512, q_stride_token=-256)) == INVALID
    assert call(lib, append=dict(table_stride=1 << 16), rotary=dict(q_out=0x600000 + (1 << 17))) == INVALID


def test_without_tokens_nothing_is_written(lib):
    assert call(lib, append=dict(tokens=0), rotary=dict(q_out=0x900000)) == OK
