"""kv_block_reads on lists that the attention accepts (no GPU needed: the
function takes CPU tensors)."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from hbfsim_b200 import kv_block_reads  # noqa: E402

CACHE = SimpleNamespace(pages=10, kv_heads=2, block_bytes=4096)


def int32(x):
    return torch.tensor(x, dtype=torch.int32)


def reads(table, blocks, counts, base=1 << 40):
    address, nbytes, op = kv_block_reads(CACHE, table, blocks, counts, base)
    assert address.dtype == torch.int64 and nbytes.dtype == torch.int32 and op.dtype == torch.uint8
    assert address.shape == nbytes.shape == op.shape and (nbytes == 4096).all() and not op.any()
    return ((address - base) // 4096).tolist()


def test_lists():
    table = int32([[3, -1, 7, 10], [0, 1, 2, 9]])
    blocks = int32([[[[2, 0], [3, 1]]], [[[3, -1], [0, 0]]]])
    counts = int32([[[2, 2]], [[1, 0]]])
    # page 10 and -1 are not in the pool; what lies behind a count is not listed
    assert reads(table, blocks, counts) == [7 * 2, 3 * 2, 9 * 2]


@pytest.mark.parametrize("bad", [-1, -7, 2, 1 << 29, -(1 << 31), (1 << 31) - 1])
def test_an_index_that_the_table_does_not_have_is_passed_over(bad):
    table = int32([[4, 5]])
    assert reads(table, int32([[[[0, bad, 1], [bad, bad, bad]]]]), int32([[[3, 3]]])) == [8, 10]


def test_nothing_listed():
    # a table without columns, as kv_select answers it; no sequences; no query tokens; empty lists
    assert reads(int32([[], []]).view(2, 0), torch.full((2, 1, 2, 3), -1, dtype=torch.int32),
                 torch.zeros((2, 1, 2), dtype=torch.int32)) == []
    for shape, width in (((0, 1, 2, 3), 4), ((2, 0, 2, 3), 4), ((2, 1, 2, 0), 4), ((0, 0, 2, 0), 0), ((0, 1, 2, 3), 0)):
        assert reads(torch.zeros((shape[0], width), dtype=torch.int32), torch.zeros(shape, dtype=torch.int32),
                     torch.full(shape[:3], 3, dtype=torch.int32)) == []


def test_views():
    table = int32([[9, 4, 5, 9], [9, 6, 7, 9]])[:, 1:3]
    every = torch.arange(2, dtype=torch.int32).expand(2, 1, 2, 2)
    assert reads(table, every, int32([2, 1])[:, None, None].expand(2, 1, 2)) == [8, 10, 9, 11, 12, 13]


def test_counts_for_all_heads_and_a_longer_table():
    """Counts that broadcast, and rows of the table behind the sequences at hand."""
    table = int32([[4, 5], [6, 7], [1, 1]])
    blocks = int32([[[[0, 1], [1, 0]]], [[[1, 0], [0, 1]]]])
    assert reads(table, blocks, int32([[[1]], [[2]]])) == [8, 11, 14, 12, 13, 15]
    with pytest.raises(ValueError):
        reads(table[:1], blocks, int32([[[1]], [[2]]]))
