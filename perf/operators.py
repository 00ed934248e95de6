"""Cases for the operators over the 8-bit paged key/value cache.

    append   new tokens' keys and values quantised into their blocks
    attend   attention of the newest tokens over all blocks of their sequence
    sparse   the same over the blocks listed for each query token and key/value head
    select   the list: a cheap score per block from bounds on its keys
    evict    blocks of least accumulated attention weight leave the block table

A cache is three tensors.  `data` (e4m3, [pages, kv heads, 2, block, dim])
holds keys then values of every (page, head); `scale` (fp32, [pages, kv heads,
2]) the power of two that each such block of values is a multiple of; `bounds`
(int8, [pages, kv heads, 2, dim]) the least and greatest stored key value of
the block per channel, rounded outwards to multiples of 4.  `table` ([seqs,
width]) maps a sequence's blocks to pages, -1 past its end.

Lengths follow from the case alone; every value follows from the seed.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3_MAX = 448.0
LOWEST, HIGHEST = -100, 120        # exponents that a block's scale may have
TOP_BYTES = 2.4e9                  # cache bytes of the largest listed case, about


def listed():
    return [
        # one token of one short chat on one head pair: the latency floor of a decode step's write
        dict(name="append one token", op="append", seqs=1, low=37, high=37, tokens=1, q_heads=8,
             kv_heads=1, dim=64, block=16, type="f16"),
        # a decode step of the paged-KV workload: 64 sequences, one token each
        dict(name="append decode step", op="append", seqs=64, low=1024, high=32768, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16"),
        # prompts entering the cache behind what their sequences hold already, ragged
        dict(name="append prompts", op="append", seqs=7, low=0, high=4001, tokens=6000,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16"),
        # the shortest decode: one sequence inside a few blocks
        dict(name="attend short", op="attend", seqs=1, low=301, high=301, tokens=1, q_heads=8,
             kv_heads=1, dim=64, block=16, type="f16", weights=True),
        # verification of 5 drafted tokens, wider blocks, eight query heads per key/value head
        dict(name="attend drafted", op="attend", seqs=8, low=700, high=9001, tokens=5, q_heads=64,
             kv_heads=8, dim=128, block=32, type="f16", weights=False),
        # one layer of a decode step of the paged-KV workload
        dict(name="attend decode step", op="attend", seqs=64, low=1024, high=32768, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", weights=True),
        # one long document: the work has to be split along its length
        dict(name="attend long", op="attend", seqs=1, low=262147, high=262147, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", weights=True),
        # the paged-KV workload's step with 128 blocks (2048 tokens) read per head
        dict(name="select decode step", op="select", seqs=64, low=1024, high=32768, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", top=128),
        dict(name="select long", op="select", seqs=1, low=262147, high=262147, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", top=128),
        dict(name="sparse decode step", op="sparse", seqs=64, low=1024, high=32768, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", top=128, weights=True),
        # every step adds weights; 20 % of the blocks of the longest sequence may stay
        dict(name="evict decode step", op="evict", seqs=64, low=1024, high=32768, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", keep=409, decay=8),
        dict(name="evict long", op="evict", seqs=1, low=262147, high=262147, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", keep=16000, decay=0),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sparse", "select", "evict"])
    dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([1, 2, 4, 4, 7, 8])
    while group * dim > 1024:
        group = rng.choice([1, 2, 4])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    block = rng.choice([16, 16, 32, 64])
    seqs = _log(rng, 1, 160)
    bytes_per_token = 2 * dim * kv_heads
    most = int(min(300000, TOP_BYTES / 1.5 / bytes_per_token / seqs))
    high = _log(rng, 1, max(1, most))
    if op == "select":
        high = max(high, 40 * block)    # fewer blocks than may be listed leave nothing to choose
    low = rng.choice([high, max(1, high // 3), 1])
    case = dict(op=op, seqs=seqs, low=low, high=high, tokens=1, q_heads=group * kv_heads,
                kv_heads=kv_heads, dim=dim, block=block, type=rng.choice(["bf16", "f16"]))
    if op == "append":
        case["low"] = rng.choice([0, low])
        case["tokens"] = rng.choice([1, _log(rng, 1, max(1, min(most, 12000 // seqs)))])
    elif op != "evict":
        case["tokens"] = rng.choice([1, 1, 2, 3, 6])
    if op in ("attend", "sparse"):
        case["weights"] = rng.choice([True, False])
    if op == "select":
        case["top"] = min(_log(rng, 6, 512), high // block // 3)
    if op == "sparse":
        case["top"] = _log(rng, 2, 512)
        each = seqs * case["tokens"] * bytes_per_token * block
        case["top"] = max(2, min(case["top"], int(TOP_BYTES / 4 / each)))
    if op == "evict":
        case["keep"] = _log(rng, 2, max(3, high // block))
        case["decay"] = rng.choice([0, 4, 8, 12])
    return case


def _spread(case):
    """Lengths between low and high, the same for every seed: multiples of the golden section."""
    at = (np.arange(case["seqs"]) * 0.6180339887498949 + 0.31) % 1.0
    return (case["low"] + np.floor(at * (case["high"] - case["low"] + 1))).astype(np.int64)


def _new_tokens(case):
    """Tokens appended per sequence: `tokens` on average, ragged where that is more than a few."""
    n, seqs = case["tokens"], case["seqs"]
    if n <= 4:
        return np.full(seqs, n, np.int64)
    at = (np.arange(seqs) * 0.7548776662466927 + 0.5) % 1.0
    return np.floor(n * (0.25 + 1.5 * at)).astype(np.int64)


def _held(case):
    """Per sequence: tokens before the call, tokens after it."""
    if case["op"] == "append":
        start = _spread(case)
        return start, start + _new_tokens(case)
    return _spread(case), _spread(case)


def _exponent(amax):
    """Least e with amax <= 448 * 2^e (448 = 0.875 * 2^9), within the limits; exact."""
    mantissa, x = torch.frexp(amax)
    e = x - 9 + (mantissa > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, LOWEST).clamp(LOWEST, HIGHEST)


def _power(e):
    """2^e in 32 bits, for -127 < e < 128."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind = "cuda", TYPES[case["type"]]
    seqs, heads, dim, block = case["seqs"], case["kv_heads"], case["dim"], case["block"]
    before, after = _held(case)
    blocks = -(-after // block)
    # an append reaches only the blocks that its tokens fall into: the others are left out here
    skip = before // block if case["op"] == "append" else 0 * blocks
    width = int(max(1, blocks.max()))
    pages = int((blocks - skip).sum()) + 3
    # blocks of a sequence lie anywhere in the pool
    order = torch.randperm(pages, generator=gen, device=dev)
    at = torch.arange(width, device=dev)
    first = torch.from_numpy(np.cumsum(blocks - skip) - blocks).to(dev)[:, None]
    blocks_dev, skip_dev = torch.from_numpy(blocks).to(dev), torch.from_numpy(skip).to(dev)[:, None]
    table = torch.where((at >= skip_dev) & (at < blocks_dev[:, None]),
                        order[(first + at).clamp(0, pages - 1)], -1).to(torch.int32)
    state = dict(case=dict(case), table=table,
                 lengths=torch.from_numpy(after).to(dev, torch.int32))
    if case["op"] == "evict":
        # attention weight of a step: a few blocks hold most of each query's
        raw = torch.rand((seqs, heads, width), generator=gen, device=dev) ** 12 + 1e-6
        raw *= (at < blocks_dev[:, None])[:, None]
        group = case["q_heads"] // heads
        state["weights"] = group * raw / raw.sum(-1, keepdim=True).clamp(min=1e-9)
        past = torch.rand((seqs, width), generator=gen, device=dev) ** 12 * (20 << 30)
        state["score"] = past.to(torch.int64) * (at < blocks_dev[:, None])
        return state
    # keys have a few strong channels, shared by all tokens of a head, and blocks differ in size
    channel = torch.exp(0.5 * torch.randn((heads, 2, 1, dim), generator=gen, device=dev))
    data = torch.empty((pages, heads, 2, block, dim), dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty((pages, heads, 2), device=dev)
    bounds = torch.empty((pages, heads, 2, dim), dtype=torch.int8, device=dev)
    chunk = max(1, (1 << 27) // (heads * 2 * block * dim))
    for a in range(0, pages, chunk):
        b = min(pages, a + chunk)
        x = torch.randn((b - a, heads, 2, block, dim), generator=gen, device=dev)
        size = torch.exp(0.6 * torch.randn((b - a, heads, 2, 1, 1), generator=gen, device=dev))
        x *= channel * size
        e = _exponent(x.abs().amax((-1, -2)))
        scale[a:b] = _power(e)
        x = _e4m3(x / scale[a:b, :, :, None, None])
        data[a:b] = x
        key = x[:, :, 0].float() / 4
        bounds[a:b, :, 0] = key.amin(-2).floor().to(torch.int8)
        bounds[a:b, :, 1] = key.amax(-2).ceil().to(torch.int8)
    state.update(data=data, scale=scale, bounds=bounds)
    # queries, keys and values are slices of one projection's output
    rows = case["q_heads"] + 2 * heads
    if case["op"] == "append":
        count = after - before
        total = int(count.sum())
        qkv = (1.5 * torch.randn((total, rows, dim), generator=gen, device=dev)).to(kind)
        state["k"] = qkv[:, case["q_heads"]:case["q_heads"] + heads]
        state["v"] = qkv[:, case["q_heads"] + heads:]
        offsets = np.concatenate([[0], np.cumsum(count)])
        state["offsets"] = torch.from_numpy(offsets).to(dev, torch.int32)
        state["start"] = torch.from_numpy(before).to(dev, torch.int32)
        # how many blocks the tokens fall into: a program knows it from its own bookkeeping
        state["touched"] = int(np.where(count > 0, (after - 1) // block - before // block + 1, 0).sum())
        return state
    qkv = (1.5 * torch.randn((seqs, case["tokens"], rows, dim), generator=gen, device=dev)).to(kind)
    state["q"] = qkv[:, :, :case["q_heads"]]
    if case["op"] == "sparse":
        # blocks at random, the newest always: what a selection looks like to the attention
        n, top = case["tokens"], case["top"]
        have = (-(-(state["lengths"].long()[:, None] - n + 1 + torch.arange(n, device=dev)) // block)).clamp(min=0)
        have = have[:, :, None].expand(seqs, n, heads)
        rank = torch.rand((seqs, n, heads, width), generator=gen, device=dev)
        rank = torch.where(at == have[..., None] - 1, 2.0, rank)
        rank = torch.where(at < have[..., None], rank, -1.0)
        best = rank.topk(min(top, width), dim=-1).indices
        if top > width:
            best = torch.cat([best, best.new_zeros(best.shape[:-1] + (top - width,))], -1)
        counts = have.clamp(max=top)
        keep = torch.arange(top, device=dev) < counts[..., None]
        best = torch.where(keep, best, width).sort(-1).values
        state["blocks"] = torch.where(keep, best, -1).to(torch.int32)
        state["counts"] = counts.to(torch.int32).contiguous()
    return state


# ---------------------------------------------------------------------------
# One pass


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _append(s):
    block = s["case"]["block"]
    data, scale, bounds, table = s["data"], s["scale"], s["bounds"], s["table"]
    start, offsets = s["start"].long(), s["offsets"].long()
    count = offsets[1:] - offsets[:-1]
    first = start // block
    many = torch.where(count > 0, (start + count - 1) // block - first + 1, 0)
    seq = torch.repeat_interleave(torch.arange(many.numel(), device=many.device), many,
                                  output_size=s["touched"])
    index = torch.arange(s["touched"], device=many.device) - (many.cumsum(0) - many)[seq] + first[seq]
    page = table[seq, index].long()
    position = index[:, None] * block + torch.arange(block, device=many.device)
    old = position < start[seq, None]
    new = ~old & (position < (start + count)[seq, None])
    token = (offsets[seq, None] + position - start[seq, None]).clamp(0, s["k"].shape[0] - 1)
    fresh = torch.stack([s["k"][token], s["v"][token]], 1).float()   # [touched, 2, block, heads, dim]
    fresh = fresh.permute(0, 3, 1, 2, 4)
    old, new = old[:, None, None, :, None], new[:, None, None, :, None]
    size = torch.where(new & fresh.isfinite(), fresh.abs(), 0).amax((-1, -2))
    need = _power(_exponent(size))
    was = scale[page]
    now = torch.where(old.any(-2).squeeze(-1), torch.maximum(was, need), need)
    held = data.view(torch.uint8)[page].view(torch.float8_e4m3fn).float()
    held = held * (was / now)[..., None, None]
    values = torch.where(new, fresh / now[..., None, None], torch.where(old, held, 0))
    values = _e4m3(values)
    data.view(torch.uint8)[page] = values.view(torch.uint8)
    scale[page] = now
    key = values[:, :, 0].float().nan_to_num() / 4
    used = (old | new)[:, :, 0]
    bounds[page] = torch.stack([torch.where(used, key, math.inf).amin(-2).floor(),
                                torch.where(used, key, -math.inf).amax(-2).ceil()], 2).to(torch.int8)
    return {"data": data, "scale": scale, "bounds": bounds}


def _softmax(s, q, key, value, see, tokens_last):
    """Weighted values, logarithm of the sum and weights of scores masked by `see`."""
    score = torch.matmul(q, key.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    score = torch.where(see, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1)
    out = torch.matmul(p, torch.where(tokens_last, value, 0))
    return out, (top + torch.log(total)).squeeze(-1), p


def _attend(s):
    c = s["case"]
    q, table, block, heads = s["q"], s["table"], c["block"], c["kv_heads"]
    seqs, n, q_heads, dim = q.shape
    group, width = q_heads // heads, table.shape[1]
    page = table.clamp(min=0).long()
    kv = s["data"].view(torch.uint8)[page].view(torch.float8_e4m3fn).float()
    kv = kv * s["scale"][page][..., None, None]              # [seqs, width, heads, 2, block, dim]
    key = kv[:, :, :, 0].transpose(1, 2).reshape(seqs, heads, width * block, dim)
    value = kv[:, :, :, 1].transpose(1, 2).reshape(seqs, heads, width * block, dim)
    rows = q.float().view(seqs, n, heads, group, dim).transpose(1, 2).reshape(seqs, heads, n * group, dim)
    position = torch.arange(width * block, device=q.device)
    last = s["lengths"].long()[:, None] - n + torch.arange(n, device=q.device)      # [seqs, n]
    see = position <= last.repeat_interleave(group, 1)[:, None, :, None]
    filled = (position < s["lengths"][:, None])[:, None, :, None]
    out, lse, p = _softmax(s, rows, key, value, see, filled)
    back = lambda x: x.view((seqs, heads, n, group) + x.shape[3:]).transpose(1, 2).reshape((seqs, n, q_heads) + x.shape[3:])  # noqa: E731
    got = {"out": back(out).to(q.dtype), "lse": back(lse)}
    if c["weights"]:
        got["weights"] = p.view(seqs, heads, n * group, width, block).sum((2, 4))
    return got


def _sparse(s):
    c = s["case"]
    q, block, heads, top = s["q"], c["block"], c["kv_heads"], c["top"]
    seqs, n, q_heads, dim = q.shape
    group, width = q_heads // heads, s["table"].shape[1]
    index = s["blocks"].long()                               # [seqs, n, heads, top]
    real = (torch.arange(top, device=q.device) < s["counts"][..., None]) & (index >= 0)
    index = torch.where(real, index, 0)
    page = torch.gather(s["table"].long(), 1, index.view(seqs, -1)).view_as(index).clamp(min=0)
    head = torch.arange(heads, device=q.device)[:, None]
    kv = s["data"].view(torch.uint8)[page, head].view(torch.float8_e4m3fn).float()
    kv = kv * s["scale"][page, head][..., None, None]        # [seqs, n, heads, top, 2, block, dim]
    key = kv[..., 0, :, :].reshape(seqs, n, heads, top * block, dim)
    value = kv[..., 1, :, :].reshape(seqs, n, heads, top * block, dim)
    rows = q.float().view(seqs, n, heads, group, dim)
    position = index[..., None] * block + torch.arange(block, device=q.device)
    last = s["lengths"].long()[:, None] - n + torch.arange(n, device=q.device)
    see = (real[..., None] & (position <= last[:, :, None, None, None])).view(seqs, n, heads, 1, top * block)
    out, lse, p = _softmax(s, rows, key, value, see, see.transpose(-1, -2))
    got = {"out": out.reshape(q.shape).to(q.dtype), "lse": lse.reshape(seqs, n, q_heads)}
    if c["weights"]:
        part = torch.where(real, p.view(seqs, n, heads, group, top, block).sum((3, 5)), 0).transpose(1, 2)
        weights = torch.zeros((seqs, heads, width), device=q.device)
        got["weights"] = weights.scatter_add_(2, index.transpose(1, 2).reshape(seqs, heads, -1),
                                              part.reshape(seqs, heads, -1))
    return got


def _select(s):
    c = s["case"]
    q, block, heads, top = s["q"], c["block"], c["kv_heads"], c["top"]
    seqs, n, q_heads, dim = q.shape
    width, dev = s["table"].shape[1], q.device
    rows = q.float().view(seqs, n, heads, q_heads // heads, dim)
    rows = torch.where(rows.isfinite(), rows, 0)
    x = torch.frexp(rows.abs().amax((-1, -2), keepdim=True)).exponent.clamp(min=LOWEST)
    whole = (rows * _power(7 - x)).round().clamp(-127, 127)
    up, down = whole.clamp(min=0).sum(3), whole.clamp(max=0).sum(3)     # [seqs, n, heads, dim]
    page = s["table"].clamp(min=0).long()
    limit = s["bounds"][page].float()                        # [seqs, width, heads, 2, dim]
    # sums of whole numbers below 2^24 for every case here: exact in 32 bits, in any order
    score = (torch.einsum("bthd,bjhd->bthj", up, limit[:, :, :, 1])
             + torch.einsum("bthd,bjhd->bthj", down, limit[:, :, :, 0]))
    score = score * s["scale"][page][..., 0].transpose(1, 2)[:, None]
    score = score.clamp(max=torch.finfo(torch.float32).max)
    have = (s["lengths"].long()[:, None] - n + torch.arange(n, device=dev)) // block + 1   # [seqs, n]
    have = have.clamp(0, width)[:, :, None, None]
    at = torch.arange(width, device=dev)
    score = torch.where((at < 1) | (at >= have - 1), math.inf, score)
    score = torch.where(at < have, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    counts = have.squeeze(-1).clamp(max=top).expand(seqs, n, heads)
    if top > width:
        order = torch.cat([order, order.new_zeros((seqs, n, heads, top - width))], -1)
    keep = torch.arange(top, device=dev) < counts[..., None]
    blocks = torch.where(keep, order, width).sort(-1).values
    return {"blocks": torch.where(keep, blocks, -1).to(torch.int32), "counts": counts.to(torch.int32)}


def _evict(s):
    c = s["case"]
    table, width, dev = s["table"], s["table"].shape[1], s["table"].device
    weight = s["weights"].nan_to_num(nan=0.0).clamp(0, 2.0 ** 20) * 2.0 ** 30
    blocks = -(-s["lengths"].long() // c["block"])[:, None]
    at = torch.arange(width, device=dev)
    here = at < blocks
    score = s["score"]
    if c["decay"]:
        score = score - (score >> c["decay"])
    score = torch.where(here, score + weight.round().to(torch.int64).sum(1), 0)
    leave = (blocks - c["keep"]).clamp(min=0)
    may = here & (at >= 1) & (at < blocks - 1)
    order = torch.where(may, score, torch.iinfo(torch.int64).max).sort(dim=-1, stable=True).indices
    gone = torch.zeros_like(here).scatter_(1, order, at < leave)
    stay = here & ~gone
    to = torch.where(stay, stay.cumsum(1) - 1, width)
    away = torch.where(gone, gone.cumsum(1) - 1, width)
    blank = torch.full((table.shape[0], width + 1), -1, dtype=table.dtype, device=dev)
    return {"score": torch.zeros((table.shape[0], width + 1), dtype=torch.int64, device=dev).scatter_(1, to, score)[:, :width],
            "table": blank.scatter(1, to, table)[:, :width],
            "lengths": (s["lengths"] - c["block"] * leave.squeeze(1)).to(torch.int32),
            "freed": blank.scatter(1, away, table)[:, :width],
            "freed_counts": leave.squeeze(1).to(torch.int32)}


_plain = {"append": _append, "attend": _attend, "sparse": _sparse, "select": _select, "evict": _evict}


def _own_append(s):
    import hbfsim_b200 as hbf
    hbf.kv_append(hbf.KvCache(s["data"], s["scale"], s["bounds"]), s["k"], s["v"], s["table"],
                  s["start"], offsets=s["offsets"])
    return {"data": s["data"], "scale": s["scale"], "bounds": s["bounds"]}


def _own_attend(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_attention(hbf.KvCache(s["data"], s["scale"], s["bounds"]), s["q"], s["table"],
                           s["lengths"], weights=s["case"]["weights"])
    return {"out": got.out, "lse": got.lse} | ({"weights": got.weights} if s["case"]["weights"] else {})


def _own_sparse(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_attention(hbf.KvCache(s["data"], s["scale"], s["bounds"]), s["q"], s["table"],
                           s["lengths"], blocks=s["blocks"], counts=s["counts"],
                           weights=s["case"]["weights"])
    return {"out": got.out, "lse": got.lse} | ({"weights": got.weights} if s["case"]["weights"] else {})


def _own_select(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_select(hbf.KvCache(s["data"], s["scale"], s["bounds"]), s["q"], s["table"],
                        s["lengths"], top=s["case"]["top"], sink=1, recent=1)
    return {"blocks": got.blocks, "counts": got.counts}


def _own_evict(s):
    import hbfsim_b200 as hbf
    c = s["case"]
    got = hbf.kv_evict(s["score"], s["weights"], s["table"], s["lengths"], keep=c["keep"],
                       block_tokens=c["block"], sink=1, recent=1, decay=c["decay"])
    return {"score": got.score, "table": got.table, "lengths": got.lengths, "freed": got.freed,
            "freed_counts": got.freed_counts}


_own = {"append": _own_append, "attend": _own_attend, "sparse": _own_sparse, "select": _own_select,
        "evict": _own_evict}


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    heads, dim, block, n = case["kv_heads"], case["dim"], case["block"], case["tokens"]
    before, after = _held(case)
    blocks = -(-after // block)
    seqs = case["seqs"]
    if case["op"] == "append":
        count = after - before
        total = int(count.sum())
        touched = int(np.where(count > 0, (after - 1) // block - before // block + 1, 0).sum())
        # the new values in, their 8-bit forms out; scales and bounds of the blocks they fall into
        return {"bytes": total * heads * dim * 2 * 3 + touched * heads * (8 + 2 * dim),
                "flops": 4 * total * heads * dim * 2}
    if case["op"] == "evict":
        held = int(blocks.sum())
        left = int(np.minimum(blocks, case["keep"]).sum())
        return {"bytes": held * (4 * heads + 8 + 4) + seqs * int(blocks.max()) * (8 + 4 + 4) + seqs * 12,
                "flops": held * heads * 3 + left}
    q_bytes = seqs * n * case["q_heads"] * dim * 2
    index = 4 * int(blocks.sum())
    # blocks that each new token may look at
    have = np.clip((after[:, None] - n + np.arange(n)) // block + 1, 0, None)
    if case["op"] == "select":
        listed_bytes = seqs * n * heads * 4 * (case["top"] + 1)
        return {"bytes": q_bytes + index + int(blocks.sum()) * heads * (2 * dim + 4) + listed_bytes,
                "flops": 4 * int(have.sum()) * heads * dim}
    out = q_bytes + seqs * n * case["q_heads"] * 4
    if case["weights"]:
        out += seqs * heads * int(blocks.max()) * 4
    if case["op"] == "attend":
        tokens = int(after.sum())
        seen = int(np.clip(after[:, None] - n + np.arange(n) + 1, 0, None).sum())
        return {"bytes": q_bytes + out + index + tokens * heads * dim * 2 + int(blocks.sum()) * heads * 8,
                "flops": 4 * seen * case["q_heads"] * dim}
    take = int(np.minimum(have, case["top"]).sum()) * heads
    # what the lists of one sequence have in common needs reading once
    once = min(take, int(blocks.sum()) * heads)
    return {"bytes": q_bytes + out + 8 * take + once * (2 * block * dim + 8),
            "flops": 4 * take * block * (case["q_heads"] // heads) * dim}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _round_e4m3(x):
    """Nearest value of 4 significant bits (ties to even), steps of 2^-9 below 2^-6, at most 448."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    step = torch.where(size / step >= 16, step * 2, torch.where(size / step < 8, step / 2, step))
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(s):
    case = s["case"]
    block = case["block"]
    start, offsets = s["start"].tolist(), s["offsets"].tolist()
    data, scale = s["data"].double(), s["scale"].double()
    table = s["table"].tolist()
    for b in range(case["seqs"]):
        done = 0
        count = offsets[b + 1] - offsets[b]
        while done < count:
            p = start[b] + done
            page, slot = table[b][p // block], p % block
            many = min(block - slot, count - done)
            a = offsets[b] + done
            for side, source in ((0, s["k"]), (1, s["v"])):
                x = source[a:a + many].double().transpose(0, 1)          # [heads, many, dim]
                size = x.abs().amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(size / 448.0)).clamp(LOWEST, HIGHEST))
                need = torch.where(size > 448.0 * need, 2 * need, need)
                need = torch.where((size <= 224.0 * need) & (need > 2.0 ** LOWEST), need / 2, need)
                now = torch.maximum(need, scale[page, :, side]) if slot else need
                old = data[page, :, side, :slot] * (scale[page, :, side] / now)[:, None, None]
                data[page, :, side] = 0
                data[page, :, side, :slot] = _round_e4m3(old)
                data[page, :, side, slot:slot + many] = _round_e4m3(x / now[:, None, None])
                scale[page, :, side] = now
            done += many
    return {"data": data, "scale": scale, "bounds": None}


def _exact_rows(q, key, value, see, dim):
    """Attention of rows [n, heads, group, dim] over key and value [n or 1, heads, tokens, dim]."""
    score = (q.double() @ key.transpose(-1, -2)) * dim ** -0.5
    score = score.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(score, -1)
    p = torch.exp(score - torch.where(lse.isinf(), 0.0, lse)[..., None]).masked_fill(~see, 0.0)
    return p @ value, lse, p


def _exact_attention(s):
    case, q = s["case"], s["q"]
    block, heads, dim = case["block"], case["kv_heads"], case["dim"]
    seqs, n, q_heads = q.shape[:3]
    group, width = q_heads // heads, s["table"].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device)
    weights = torch.zeros((seqs, heads, width), dtype=torch.float64, device=q.device)
    lengths = s["lengths"].tolist()
    for b in range(seqs):
        for t in range(n):
            last = lengths[b] - n + t
            for h in range(heads):
                if "blocks" in s:
                    many = int(s["counts"][b, t, h])
                    index = s["blocks"][b, t, h, :many].long()
                else:
                    index = torch.arange(-(-lengths[b] // block), device=q.device)
                page = s["table"][b].long()[index]
                kv = s["data"].view(torch.uint8)[page, h].view(torch.float8_e4m3fn).double()
                kv = kv * s["scale"][page, h].double()[..., None, None]      # [blocks, 2, block, dim]
                see = (index[:, None] * block + torch.arange(block, device=q.device) <= last).view(-1)
                rows = q[b, t, h * group:(h + 1) * group]
                o, m, p = _exact_rows(rows, kv[:, 0].reshape(-1, dim), kv[:, 1].reshape(-1, dim), see, dim)
                out[b, t, h * group:(h + 1) * group] = o
                lse[b, t, h * group:(h + 1) * group] = m
                weights[b, h].index_add_(0, index, p.view(group, -1, block).sum((0, 2)))
    got = {"out": out, "lse": lse}
    return got | ({"weights": weights} if case["weights"] else {})


def exact(case, seed):
    if case["op"] in ("select", "evict"):
        return None                     # whole numbers, which the plain form gives exactly
    if case["seqs"] * case["tokens"] * case["kv_heads"] > 6000 and case["op"] != "append":
        return None                     # one small product at a time: too many of them
    if case["op"] == "append" and case["seqs"] * case["tokens"] // case["block"] > 6000:
        return None
    return (_exact_append if case["op"] == "append" else _exact_attention)(prepare(case, seed))
