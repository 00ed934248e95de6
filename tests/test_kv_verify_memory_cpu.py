"""kv_verify turns down outputs that lie in the inputs' memory or in each other's, before any device
work (no GPU needed)."""
import ctypes

import pytest

from hbfsim_b200 import _lib, build
from test_kv_cpu import INVALID, OK

ref = ctypes.byref


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def verify(**over):
    """2 sequences of 3 drafts over 100 fp32 values, every array 64 KB from the next."""
    given = dict(struct_size=ctypes.sizeof(_lib.KvVerifyBatchV1), version=1, type=2, seqs=2, drafts=3, vocab=100,
                 target=0x100000, target_stride_seq=400, target_stride_token=100, draft=0x110000,
                 draft_stride_seq=300, draft_stride_token=100, tokens=0x120000, accept=0x130000, sample=0x140000,
                 counts=0x150000, lengths=0x160000, accepted=0x170000, tokens_out=0x180000, lengths_out=0x190000)
    return _lib.KvVerifyBatchV1(**{**given, **over})


@pytest.mark.parametrize("over", [
    # in an input's memory
    dict(tokens_out=0x120000), dict(tokens_out=0x120000 + 20), dict(tokens_out=0x120000 - 28),
    dict(tokens_out=0x130000 + 4), dict(tokens_out=0x140000), dict(tokens_out=0x150000), dict(tokens_out=0x160000),
    dict(accepted=0x120000), dict(accepted=0x130000 + 20), dict(accepted=0x140000), dict(accepted=0x160000),
    dict(lengths_out=0x120000), dict(lengths_out=0x140000 - 4), dict(lengths_out=0x150000),
    # in place, but not element by element
    dict(accepted=0x150000 + 4), dict(accepted=0x150000 - 4), dict(lengths_out=0x160000 + 4),
    # in each other's
    dict(accepted=0x180000), dict(accepted=0x180000 + 28), dict(lengths_out=0x180000 - 4), dict(accepted=0x190000),
    dict(accepted=0x160000, lengths_out=0x160000), dict(accepted=0x150000, lengths_out=0x150000, lengths=0x150000),
    # in the probabilities: the first and the last of them, rows in descending order
    dict(accepted=0x100000), dict(tokens_out=0x100000 + 799 * 4), dict(lengths_out=0x110000 + 599 * 4),
    dict(accepted=0x100000 - 400 * 4, target_stride_seq=-400), dict(accepted=0x110000 - 200 * 4, draft_stride_token=-100)])
def test_outputs_in_other_memory_are_refused(lib, over):
    assert lib.hbfsim_kv_verify_v1(ref(verify(**over)), None) == INVALID


@pytest.mark.parametrize("over", [dict(tokens=None), dict(accept=None), dict(sample=None), dict(target=None),
                                  dict(accepted=None), dict(tokens_out=None), dict(lengths=None), dict(sample=0x140002),
                                  dict(counts=0x150001), dict(tokens_out=0x180002), dict(vocab=0), dict(seqs=65537)])
def test_refusals_with_every_array_apart(lib, over):
    assert lib.hbfsim_kv_verify_v1(ref(verify(**over)), None) == INVALID


def test_no_sequence_is_no_race(lib):
    assert lib.hbfsim_kv_verify_v1(ref(verify(seqs=0, accepted=0x100000, tokens_out=0x100000)), None) == OK
