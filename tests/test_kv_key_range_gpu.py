"""Block lists and evictions whose scores reach the ends of their type: the
search for the last key narrows a range that may not wrap.  Results are equal
to the definitions' (oracle/kv_oracle.py)."""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import assert_lists, int32, to_gpu, torch_

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("blocks,seqs", [(17000, 1), (17000, 160), (300000, 1)])
@pytest.mark.parametrize("share", [0.1, 0.5, 0.8, 0.999])
def test_select_scores_near_the_largest_floats(blocks, seqs, share):
    """One channel of the query counts: scores are bound * 2^120, some 1.3e38 at most."""
    torch = torch_()
    from hbfsim_b200 import kv_select
    rng = np.random.default_rng(blocks)
    dim, block, pages = 64, 16, 400
    cache = {"data": np.zeros((pages, 1, 2, block, dim), np.uint8), "scale": np.full((pages, 1, 2), 2.0 ** 114),
             "bounds": np.zeros((pages, 1, 2, dim), np.int8)}
    # page 0 holds the greatest, page 1 the least; the scales add values between
    cache["bounds"][:, 0, 1, 5] = np.concatenate([[100, -100], rng.integers(-100, 101, pages - 2)])
    cache["scale"][2:, 0, 0] *= 2.0 ** -rng.integers(0, 4, pages - 2)
    table = rng.integers(0, pages, (1, blocks)).astype(np.int32)
    q = np.zeros((1, 1, 1, dim))
    q[..., 5] = 1.0
    top = int(share * blocks)
    lists = ko.select(cache, q, table, [blocks * block], top, 1, 1)
    got = kv_select(to_gpu(cache), torch.from_numpy(q).to(torch.bfloat16).cuda().expand(seqs, 1, 1, dim),
                    int32(table).expand(seqs, blocks), int32([blocks * block] * seqs), top)
    assert_lists(type(got)(got.blocks[:1], got.counts[:1]), lists)
    assert (got.blocks == got.blocks[:1]).all() and (got.counts == got.counts[:1]).all()


@pytest.mark.parametrize("blocks,seqs", [(100, 3), (3000, 200), (9000, 1), (60000, 1), (250000, 1)])
@pytest.mark.parametrize("low,high,share", [(5, (1 << 63) - 1, 0.75), (-(1 << 63), (1 << 63) - 1, 0.9),
                                            (-(1 << 63), (1 << 63) - 1, 0.2), (1 << 62, (1 << 63) - 1, 0.6)])
def test_evict_scores_near_the_largest_integers(blocks, seqs, low, high, share):
    """Half of the scores near the least of a range, half near the greatest."""
    torch = torch_()
    from hbfsim_b200 import kv_evict
    rng = np.random.default_rng(blocks + seqs)
    near = rng.integers(0, 1 << 56, blocks)
    near[rng.random(blocks) < 0.1] = 7  # equal ones
    score = np.where(rng.random(blocks) < 0.5, low + near, high - near).astype(np.int64)[None]
    table = rng.permutation(blocks).astype(np.int32)[None]
    weights = np.zeros((1, 1, blocks), np.float32)
    keep = max(2, blocks - int(share * blocks))
    want = ko.evict(score, weights, table, [blocks * 16], keep, 16, 1, 1, 0)
    cuda = lambda x: torch.from_numpy(np.repeat(x, seqs, 0)).cuda()  # noqa: E731
    got = kv_evict(cuda(score), cuda(weights), cuda(table), int32([blocks * 16] * seqs), keep)
    for a, b, name in zip(got, want, got._fields):
        assert np.array_equal(a.cpu().numpy(), np.repeat(b, seqs, 0)), name
