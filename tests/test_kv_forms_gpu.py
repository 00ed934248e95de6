"""The attention over the 8-bit paged cache takes one of several forms by a
call's sizes (hbfsim_b200/csrc/kv_plan.h).  Every test here says which one it
means and checks that it got it: rows shared out among thread blocks and joined
by a second kernel (the call then needs a workspace), or finished by the thread
blocks that sum them, of 4 or 8 warps, alone or in teams.  Bounds are those of
test_kv_gpu.py."""
import numpy as np
import pytest

from test_kv_gpu import ATTENDS, attend_and_check, int32, make_table, random_cache, to_gpu, torch_, type_of
from test_kv_scales_gpu import splits

pytestmark = pytest.mark.gpu


def lists_of(rng, lengths, tokens, heads, block, share=1.0):
    return [[[[int(j) for j in rng.permutation(-(-n // block)) if rng.random() < share] for _ in range(heads)]
             for _ in range(tokens)] for n in lengths]


def check(small, q, table, lengths, split, lists=None, weights=True):
    """One call twice, in the form that is meant; the same bits both times."""
    torch = torch_()
    gpu = to_gpu(small)
    shape = None
    if lists is not None:
        top = max(1, max((len(x) for b in lists for t in b for x in t), default=1)) + 1
        shape = np.zeros(q.shape[:2] + (gpu.kv_heads, top))
    assert splits(gpu, q, int32(table), int32(lengths), shape, weights) == split, "not the form that is meant"
    got = attend_and_check(small, q, table, lengths, lists, gpu=gpu, weights=weights)
    again = attend_and_check(small, q, table, lengths, lists, gpu=gpu, weights=weights)
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)
    return got


@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("dim,block,heads,group,tokens,kind,lengths", ATTENDS + [
    (128, 16, 2, 8, 3, "bf16", [300, 2, 77, 1500]),   # 24 rows of 128 channels
    (128, 32, 1, 24, 1, "f16", [1, 900]),
    (64, 16, 1, 6, 4, "bf16", [0, 257]), (256, 16, 1, 8, 1, "bf16", [700]), (256, 64, 2, 1, 1, "f16", [65, 64])])
def test_shared_out_and_joined(dim, block, heads, group, tokens, kind, lengths, weights):
    torch = torch_()
    rng = np.random.default_rng(dim + block + heads + group + tokens)
    pages = int(sum(-(-n // block) for n in lengths)) + 2
    cache = random_cache(rng, pages, heads, block, dim)
    # room for more tiles than teams of thread blocks may finish
    table = make_table(rng, lengths, block, pages, extra=20000 // block)
    for b, n in enumerate(lengths):
        if n % block:
            cache["data"][table[b, n // block], :, :, n % block:] = 0x7f
    x = 1.5 * rng.standard_normal((len(lengths), tokens, (group + 1) * heads, dim))
    q = torch.from_numpy(x).to(type_of(kind)).cuda()[:, :, heads:]
    check(cache, q, table, lengths, True, weights=weights)


@pytest.mark.parametrize("dim,block,heads,group,kind,blocks,seqs", [
    (128, 16, 2, 4, "bf16", 700, 5), (64, 32, 1, 24, "f16", 300, 3), (256, 16, 2, 9, "bf16", 200, 3)])
def test_long_lists_shared_out_and_joined(dim, block, heads, group, kind, blocks, seqs):
    """Two query tokens with a list each: weights of both, by segments of one (sequence, head)."""
    torch = torch_()
    rng = np.random.default_rng(blocks)
    small = random_cache(rng, 40, heads, block, dim)
    table = rng.integers(0, 40, (seqs, blocks)).astype(np.int32)
    lengths = [int(x) for x in rng.integers(1, blocks * block, seqs)]
    q = torch.from_numpy(rng.standard_normal((seqs, 2, heads * group, dim))).to(type_of(kind)).cuda()
    lists = lists_of(rng, lengths, 2, heads, block, 0.5)
    lists[0][1][0] = []
    check(small, q, table, lengths, True, lists)


@pytest.mark.parametrize("group,tokens,kind", [(8, 5, "f16"), (8, 5, "bf16"), (20, 2, "bf16")])
@pytest.mark.parametrize("weights,width", [(False, 60), (True, 900)])
def test_segments_that_several_thread_blocks_join(group, tokens, kind, weights, width):
    """8 sequences of 8 heads with 40 rows each: three segments to a pair, more thread blocks of
    the joining kernel than segments, so that each joins a slice of one."""
    torch = torch_()
    rng = np.random.default_rng(group + tokens + width)
    seqs, heads, dim, block = 8, 8, 128, 32
    small = random_cache(rng, 30, heads, block, dim)
    table = rng.integers(0, 30, (seqs, width)).astype(np.int32)
    lengths = [0, 1, 1000, 31, 700, 64, 333, 5]
    q = torch.from_numpy(rng.standard_normal((seqs, tokens, heads * group, dim))).to(type_of(kind)).cuda()
    check(small, q, table, lengths, True, weights=weights)


@pytest.mark.parametrize("dim,group,tokens", [(64, 2, 3), (64, 4, 4), (64, 5, 4), (128, 1, 6), (128, 8, 2), (128, 8, 3),
                                              (128, 8, 5), (256, 2, 4), (256, 5, 3)])
@pytest.mark.parametrize("apart", [0, 40])
@pytest.mark.parametrize("split", [True, False])
def test_nan_stays_in_the_rows_that_see_it(dim, group, tokens, apart, split):
    """A key and a value that are NaN at the last positions, in both forms, and with value scales
    that are far apart (2^apart): earlier query tokens must not meet them, later ones do."""
    torch = torch_()
    from hbfsim_b200 import kv_attention
    rng = np.random.default_rng(dim + group)
    block, heads, n = 16, 2, 340
    pages = -(-n // block)
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, [n], block, pages, extra=20000 // block if split else 0)
    cache["scale"][table[0, 2::3][table[0, 2::3] >= 0], :, 1] *= 2.0 ** -apart
    q = torch.from_numpy(rng.standard_normal((1, tokens, heads * group, dim))).to(torch.bfloat16).cuda()
    eights = -(-group * tokens // 8)
    one_pass = eights <= 2 or (eights == 3 and dim < 256)
    weights = split and one_pass  # without weights several passes may be finished whole too
    tab, lens = int32(table), int32([n])
    assert splits(to_gpu(cache), q, tab, lens, None, weights) == split, "not the form that is meant"
    clean = attend_and_check(cache, q, table, [n], weights=weights)
    for side in (0, 1):
        for position in (n - 1, n - 2, n - tokens):
            bad = {k: v.copy() for k, v in cache.items()}
            bad["data"][table[0, position // block], 1, side, position % block] = 0x7f
            got = kv_attention(to_gpu(bad), q, tab, lens, weights=weights)
            sees = torch.arange(n - tokens, n, device="cuda") >= position
            hit = torch.arange(heads * group, device="cuda") >= group  # the second head's queries
            rows = sees[:, None] & hit
            assert torch.isnan(got.out[0, rows]).all()
            assert torch.equal(got.out[0, ~rows], clean.out[0, ~rows])
            assert torch.equal(got.lse[0, ~rows], clean.lse[0, ~rows])
            assert torch.isnan(got.lse[0, rows]).all() == (side == 0)
            if weights:
                assert torch.equal(got.weights[0, 0], clean.weights[0, 0])


WHOLE = [  # dim, block, heads, group, kind, seqs, blocks: more (sequence, head) pairs than SMs: 4 warps
    (64, 16, 8, 4, "bf16", 25, 60), (64, 32, 8, 16, "f16", 25, 16), (64, 16, 8, 24, "bf16", 25, 30),
    (128, 16, 8, 8, "f16", 25, 60), (128, 64, 8, 12, "bf16", 25, 8), (128, 16, 8, 20, "f16", 25, 32),
    (256, 16, 8, 8, "bf16", 25, 50), (256, 32, 8, 11, "f16", 25, 16),
    # fewer: 8 warps, and teams of them
    (64, 16, 2, 16, "bf16", 3, 60), (64, 16, 2, 20, "f16", 3, 200), (128, 16, 2, 12, "bf16", 3, 50),
    (128, 32, 2, 24, "f16", 3, 90), (256, 16, 2, 7, "bf16", 3, 60), (256, 64, 2, 16, "f16", 3, 40)]


@pytest.mark.parametrize("dim,block,heads,group,kind,seqs,blocks", WHOLE)
def test_finished_where_they_are_summed(dim, block, heads, group, kind, seqs, blocks):
    torch = torch_()
    rng = np.random.default_rng(dim + group + blocks)
    small = random_cache(rng, 30, heads, block, dim)
    table = rng.integers(0, 30, (seqs, blocks)).astype(np.int32)
    table[rng.random(table.shape) < 0.03] = -1
    lengths = [blocks * block, 0, 1] + [int(x) for x in rng.integers(0, blocks * block, seqs - 3)]
    q = torch.from_numpy(rng.standard_normal((seqs, 1, heads * group, dim))).to(type_of(kind)).cuda()
    check(small, q, table, lengths, False)
    check(small, q, table, lengths, False, weights=False)
