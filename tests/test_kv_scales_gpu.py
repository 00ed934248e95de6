"""Attention over the 8-bit paged cache where the blocks' value scales are far
apart: a block counts by its weight, whatever scales its neighbours have.

The bound on an output is that of test_kv_gpu.py without its term in the
largest value in view: the probabilities keep a relative precision of 2^-11,
so an output is off by that share of its mass (softmax mean of |values|), by
2 d + 2^-20 from the scores and the exponentials (d = 2^-19 * reach) and by
the output type's half unit.  Probabilities may be held in f16 among blocks
whose scales are within 2^10 of each other, the largest at 2^10 or more, so
that each is off by 2^-35 of the largest probability times scale among those
of one size of scale: tokens * 2^-35 * 448 * largest in all.
"""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import int32, make_table, random_cache, to_gpu, torch_, type_of

pytestmark = pytest.mark.gpu


def splits(gpu, q, table, lengths, lists, weights):
    """Whether the call shares its rows out and joins them: it then needs a workspace."""
    from hbfsim_b200 import _lib, kv
    query = kv._query(gpu, q, table, lengths)[0]
    top, at = (lists.shape[3], 16) if lists is not None else (0, 0)
    args = kv._ATTENTION.pack(kv._ATTENTION.size, 1, 0.1, top, at, at, 16, 16, 16 if weights else 0, 0, 0)
    return _lib.load().hbfsim_kv_attention_workspace_v1(gpu._packed, query, args) > 0


def encode_at(x):
    return ko.encode(np.asarray(x, np.float64))


def build(rng, mode, dim, block, group, tokens, kind, blocks, up, down, heads=2):
    """One sequence; `loud` blocks have value scales 2^(up - down) above the others.  mode:
    negligible  scores of the loud blocks are 176 sqrt(dim / 64) below the others'
    rows        the same for the even query heads; the odd ones see little else
    zero        scores like the others', every value 0
    unseen      the last block: the values that the first token sees are 0"""
    torch = torch_()
    n = blocks * block - 3
    cache = random_cache(rng, blocks, heads, block, dim)
    table = make_table(rng, [n], block, blocks)
    loud = table[0, [blocks - 1] if mode == "unseen" else [0, blocks // 2, blocks // 2 + 1, blocks - 1]]
    quiet = np.setdiff1d(np.arange(blocks), loud)
    sign = rng.choice([-1.0, 1.0], dim)
    cache["scale"][quiet, :, 0] = 1.0
    cache["data"][quiet, :, 0] = encode_at(0.5 * rng.standard_normal((quiet.size, heads, block, dim)))
    cache["scale"][loud, :, 0] = 1.0
    near = 0.5 * rng.standard_normal((loud.size, heads, block, dim))
    cache["data"][loud, :, 0] = encode_at(near if mode in ("zero", "unseen") else -11 * sign + 0 * near)
    cache["scale"][quiet, :, 1] *= 2.0 ** down
    cache["scale"][loud, :, 1] *= 2.0 ** up
    if mode == "zero":
        cache["data"][loud, :, 1] = 0
    if mode == "unseen":
        cache["data"][loud, :, 1, :block - 3 - tokens + 1] = 0
    q = 2 * sign + 0.3 * rng.standard_normal((1, tokens, heads * group, dim))
    if mode == "rows":
        q[:, :, 1::2] *= -1
    q = torch.from_numpy(q).to(type_of(kind)).cuda()
    return cache, table, n, q, loud


def attend_and_check(cache, q, table, n, loud, lists=None, weights=True, split=None):
    torch = torch_()
    from hbfsim_b200 import kv_attention
    gpu = to_gpu(cache)
    blocks = counts = None
    tokens, heads = q.shape[1], gpu.kv_heads
    if lists is not None:
        blocks = int32(np.broadcast_to(lists, (1, tokens, heads, len(lists))))
        counts = int32(np.full((1, tokens, heads), len(lists)))
    tab, lens = int32(table), int32([n])
    if split is not None:
        assert splits(gpu, q, tab, lens, blocks, weights) == split, "not the form that is meant"
    got = kv_attention(gpu, q, tab, lens, blocks=blocks, counts=counts, weights=weights)
    torch.cuda.synchronize()
    D = q.shape[3]
    given = None if lists is None else [[[list(lists)] * heads] * tokens]
    args = (q.double().cpu().numpy(), table, [n], D ** -0.5, given)
    out, lse, mass_w, mass, reach, _ = ko.attention(cache, *args)
    # probability times scale at most, among the blocks of one size of scale
    top = np.zeros(reach.shape)
    for pages in (loud, np.setdiff1d(np.arange(gpu.pages), loud)):
        part = {k: v.copy() for k, v in cache.items()}
        part["data"][:, :, 1] = 0
        part["data"][pages, :, 1] = 0x38  # 1.0: the mass is the mean of the scales
        top = np.maximum(top, np.where(np.isin(pages, loud).all(), 0, ko.attention(part, *args)[3].max(-1)))
    d = 2.0 ** -19 * reach
    unit, least = (2.0 ** -8, 2.0 ** -133) if q.dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -24)
    tol = (unit * np.abs(out) + (2.0 ** -11 + 2 * d + 2.0 ** -20)[..., None] * mass * (1 + unit)
           + n * 2.0 ** -35 * 448 * top[..., None] + least)
    go = got.out.double().cpu().numpy()
    most = torch.finfo(q.dtype).max
    past = np.abs(out) + tol > most
    assert (np.isfinite(go) | past).all()
    off = np.abs(np.clip(go, -most, most) - np.clip(out, -most, most))
    assert (off <= tol).all(), f"out: {np.nanmax(off / tol)} times the bound"
    gl = got.lse.double().cpu().numpy()
    assert (np.abs(gl - lse) <= d + 2.0 ** -20 * (1 + np.abs(lse))).all()
    if weights:
        gw = got.weights.double().cpu().numpy()
        assert (np.abs(gw - mass_w) <= mass_w * (2 * d.max() + 2.0 ** -19) + 1e-30).all()


FORMS = [  # dim, block, group, tokens, blocks, blocks of room behind, split
    (64, 16, 4, 1, 30, 0, False),      # finished by one thread block
    (128, 16, 8, 1, 100, 0, False),    # by a team of them
    (128, 16, 4, 1, 60, 2500, True),   # shared out and joined
    (64, 32, 8, 5, 23, 0, True),       # several row tiles
    (128, 16, 6, 4, 40, 2500, True),   # 24 rows at once
    (256, 16, 3, 4, 31, 0, False),
    (256, 64, 5, 3, 20, 400, True)]
SCALES = [("bf16", 0, 0), ("bf16", 8, -8), ("bf16", 14, -14), ("bf16", 30, -30), ("bf16", 100, -90),
          ("f16", 24, 0), ("f16", 60, 0)]


@pytest.mark.parametrize("dim,block,group,tokens,blocks,extra,split", FORMS)
@pytest.mark.parametrize("mode", ["negligible", "rows", "zero", "unseen"])
def test_value_scales_far_apart(dim, block, group, tokens, blocks, extra, split, mode):
    for kind, up, down in SCALES:
        rng = np.random.default_rng(dim + blocks + up)
        cache, table, n, q, loud = build(rng, mode, dim, block, group, tokens, kind, blocks, up, down)
        wide = np.concatenate([table, np.full((1, extra), -1, np.int32)], 1)
        attend_and_check(cache, q, wide, n, loud, split=split)
        if tokens == 1:  # loud blocks first, last and among the others
            rest = [j for j in range(blocks) if table[0, j] not in loud]
            at = [j for j in range(blocks) if table[0, j] in loud]
            for lists in (at + rest, rest + at, list(rng.permutation(blocks))):
                attend_and_check(cache, q, wide, n, loud, lists=lists)


def test_values_near_the_largest():
    """Sums of values that 32 bits cannot hold, of a mean that they can."""
    torch = torch_()
    rng = np.random.default_rng(3)
    dim, block, heads, blocks = 64, 16, 1, 60
    for extra, split in ((0, False), (2500, True)):
        cache = random_cache(rng, blocks, heads, block, dim)
        cache["scale"][:, :, 1] = 2.0 ** 118
        cache["data"][:, :, 1] = encode_at(448 * rng.random((blocks, heads, block, dim)))
        table = make_table(rng, [blocks * block], block, blocks, extra=extra)
        q = torch.from_numpy(0.1 * rng.standard_normal((1, 1, 4, dim))).to(torch.bfloat16).cuda()
        attend_and_check(cache, q, table, blocks * block, np.array([], int), split=split)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim,extra,seqs,split", [(64, 0, 40, False), (128, 90, 4, False), (256, 10, 4, False),
                                                  (64, 20000, 40, True), (128, 20000, 40, True)])
def test_a_row_of_one_token_is_its_value(dim, extra, seqs, split, kind):
    """The one probability is 1 whatever the score: the output is the stored value, bit for bit."""
    torch = torch_()
    from hbfsim_b200 import kv_attention
    rng = np.random.default_rng(dim + extra)
    block, heads, group = 16, 2, 4
    cache = random_cache(rng, seqs, heads, block, dim)
    cache["scale"][:, :, 1] = 2.0 ** rng.integers(-9, 3, (seqs, heads))
    table = make_table(rng, [1] * seqs, block, seqs, extra=extra)
    q = torch.from_numpy(3 * rng.standard_normal((seqs, 1, heads * group, dim))).to(type_of(kind)).cuda()
    gpu, tab, lens = to_gpu(cache), int32(table), int32([1] * seqs)
    assert splits(gpu, q, tab, lens, None, True) == split, "not the form that is meant"
    got = kv_attention(gpu, q, tab, lens, weights=True)
    value = ko.E4M3[cache["data"][table[:, 0], :, 1, 0]] * cache["scale"][table[:, 0], :, 1][..., None]
    want = np.repeat(value, group, 1)[:, None]
    assert np.array_equal(got.out.double().cpu().numpy(), want)
    assert np.abs(got.weights[:, :, 0].double().cpu().numpy() - group).max() <= 2.0 ** -18
    assert not got.weights[:, :, 1:].any()
