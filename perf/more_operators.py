"""Cases for what surrounds attention on the 8-bit paged key/value cache.

    rotary   queries and keys rotated by positions on several axes, the keys
             and values quantised into the cache's blocks
    verify   drafted tokens accepted or not, and the token that comes next
    resize   every sequence gets or gives back pages, shared blocks are parted
    fork     sequences go on as children of others; pages are counted
    copy     pages' contents to other pages
    compact  pages in use move to the front of the pool

A cache is three tensors.  `data` (e4m3, [pages, kv heads, 2, block, dim])
holds keys then values of every (page, head); `scale` (fp32, [pages, kv heads,
2]) the power of two that each such block of values is a multiple of; `bounds`
(int8, [pages, kv heads, 2, dim]) the least and greatest stored key value of
the block per channel, rounded outwards to multiples of 4 and divided by 4.
`table` ([seqs, width]) maps a sequence's blocks to pages, -1 past its end;
`refs` ([pages]) counts the entries that name a page, which is free while its
count is not positive.

Lengths follow from the case alone; every value follows from the seed.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3_MAX = 448.0
LOWEST, HIGHEST = -100, 120        # exponents that a block's scale may have
PROMPT_TOKENS = 31668              # new tokens of the largest listed rotary case, about
VERIFY_VALUES = 64 * 5 * 131072    # target probabilities of the largest listed verification
COPY_BYTES = 1.0e9                 # page bytes of the largest listed copy, about


def listed():
    return [
        # a decode step of the paged-KV workload: 64 sequences, one token each, positions in
        # time, height and width as a model of text and images has them
        dict(name="rotary decode step", op="rotary", seqs=64, low=1024, high=32768, tokens=1,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", rotated=128, axes=3,
             neighbours=False),
        # prompts with images entering the cache behind what their sequences hold already, ragged
        dict(name="rotary prompts", op="rotary", seqs=7, low=0, high=4001, tokens=6000,
             q_heads=32, kv_heads=8, dim=128, block=16, type="bf16", rotated=128, axes=3,
             neighbours=False),
        # one chat on a small vocabulary, drafts without probabilities (looked up in the prompt)
        dict(name="verify one chat", op="verify", seqs=1, tokens=3, vocab=32768, type="f32",
             draft=False),
        # the drafted step: 4 drafted tokens of 64 sequences, a draft model's probabilities
        dict(name="verify drafted step", op="verify", seqs=64, tokens=4, vocab=131072, type="f32",
             draft=True),
        # before a step of the paged-KV workload: beams just forked part their last blocks, some
        # sequences begin a block, evicted pages come back
        dict(name="resize decode step", op="resize", seqs=64, low=1024, high=32768, tokens=5,
             block=16, beams=4, mix=False, spare=0.05, evicted=2),
        # a large server's pool: a third of the rows finish, a third step, a third take prompts
        dict(name="resize server", op="resize", seqs=510, low=8000, high=65536, tokens=1,
             block=16, beams=1, mix=True, spare=0.1, evicted=0),
        # beams of 16 requests are reordered
        dict(name="fork beams", op="fork", seqs=64, low=1024, high=32768, rows=64, block=16,
             beams=4),
        # a few long documents answered many times over
        dict(name="fork documents", op="fork", seqs=4, low=200000, high=262147, rows=256,
             block=16, beams=1),
        # copy on write of one layer: a partly filled page for each sequence
        dict(name="copy shared blocks", op="copy", moves=64, pages=2048, kv_heads=8, dim=128,
             block=16),
        # one layer's moves of a compaction: a gigabyte
        dict(name="copy compaction", op="copy", moves=28000, pages=60000, kv_heads=8, dim=128,
             block=16),
        # a small pool after its sequences came and went
        dict(name="compact small pool", op="compact", seqs=16, low=200, high=4000, block=16,
             gone=0.5),
        # the server's pool before it shrinks
        dict(name="compact server", op="compact", seqs=512, low=8000, high=65536, block=16,
             gone=0.4),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "verify", "verify", "resize", "fork", "copy", "compact"])
    if op == "verify":
        n = rng.choice([1, 1, 2, 3, 5, 7, 15])
        seqs = _log(rng, 1, 300)
        return dict(op=op, seqs=seqs, tokens=n,
                    vocab=_log(rng, 100, min(260000, max(200, VERIFY_VALUES // (seqs * (n + 1))))),
                    type=rng.choice(["f32", "f32", "bf16", "f16"]), draft=rng.choice([True, False]))
    if op in ("rotary", "copy"):
        dim, kv_heads, block = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8, 8]), rng.choice([16, 16, 32, 64])
    if op == "copy":
        page = 2 * kv_heads * dim * (block + 1)
        pages = _log(rng, 4, int(COPY_BYTES / page))
        return dict(op=op, moves=_log(rng, 1, pages // 2), pages=pages, kv_heads=kv_heads, dim=dim, block=block)
    if op == "rotary":
        group = rng.choice([1, 2, 4, 4, 7, 8])
        seqs = _log(rng, 1, 160)
        # as many values as the largest listed case at most
        most = max(1, PROMPT_TOKENS * 48 * 128 // ((group + 2) * kv_heads * dim * seqs))
        high = _log(rng, 1, 40000)
        return dict(op=op, seqs=seqs, low=rng.choice([0, high // 3, high]), high=high,
                    tokens=rng.choice([1, _log(rng, 1, max(1, min(most // 2, 6000)))]),
                    q_heads=group * kv_heads, kv_heads=kv_heads, dim=dim, block=block,
                    type=rng.choice(["bf16", "f16"]), rotated=rng.choice([dim, dim, dim // 2, dim // 4]),
                    axes=rng.choice([1, 3, 3, 4]), neighbours=rng.choice([False, False, True]))
    block = rng.choice([16, 16, 32, 64])
    beams = rng.choice([1, 2, 4, 4])
    seqs = beams * _log(rng, 1, 300 // beams)
    high = _log(rng, 1, max(1, min(262147, 16000000 // seqs)))
    case = dict(op=op, seqs=seqs, low=rng.choice([high, max(1, high // 3), 1]), high=high, block=block)
    if op == "compact":
        return case | dict(gone=rng.choice([0.02, 0.3, 0.5, 0.9]))
    case["beams"] = beams
    if op == "fork":
        return case | dict(rows=_log(rng, 1, max(1, min(300, 16000000 // high))))
    return case | dict(tokens=rng.choice([1, 1, 5, 300]), mix=rng.choice([False, False, True]),
                       spare=rng.choice([0.0, 0.05, 0.3]), evicted=rng.choice([0, 2]))


def _spread(low, high, count):
    """Values between low and high, the same for every seed: multiples of the golden section."""
    at = (np.arange(count) * 0.6180339887498949 + 0.31) % 1.0
    return (low + np.floor(at * (high - low + 1))).astype(np.int64)


def _new_tokens(case):
    """Tokens appended per sequence: `tokens` on average, ragged where that is more than a few."""
    n, seqs = case["tokens"], case["seqs"]
    if n <= 4:
        return np.full(seqs, n, np.int64)
    at = (np.arange(seqs) * 0.7548776662466927 + 0.5) % 1.0
    return np.floor(n * (0.25 + 1.5 * at)).astype(np.int64)


def _lengths(case):
    """Tokens that each row of a pool's table holds: beams of one request are equally long."""
    beams = case.get("beams", 1)
    return np.repeat(_spread(case["low"], case["high"], -(-case["seqs"] // beams)), beams)[:case["seqs"]]


def _wanted(case):
    """Per row of a resize: tokens held, tokens wanted."""
    held = _lengths(case)
    want = held + case["tokens"]
    if case["mix"]:
        kind = np.arange(case["seqs"]) // case["beams"] % 3      # 0 finished, 1 a step, 2 a prompt that enters
        want = np.where(kind == 0, 0, np.where(kind == 2, held, want))
        held = np.where(kind == 2, 0, held)
    return held, want


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


def _cache(gen, pages, heads, block, dim):
    """Pages of keys and values: a few strong key channels, pages of different size."""
    dev = "cuda"
    channel = torch.exp(0.5 * torch.randn((heads, 2, 1, dim), generator=gen, device=dev))
    data = torch.empty((pages, heads, 2, block, dim), dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty((pages, heads, 2), device=dev)
    bounds = torch.empty((pages, heads, 2, dim), dtype=torch.int8, device=dev)
    chunk = max(1, (1 << 27) // (heads * 2 * block * dim))
    for a in range(0, pages, chunk):
        b = min(pages, a + chunk)
        x = torch.randn((b - a, heads, 2, block, dim), generator=gen, device=dev)
        x *= channel * torch.exp(0.6 * torch.randn((b - a, heads, 2, 1, 1), generator=gen, device=dev))
        scale[a:b] = _power(_exponent(x.abs().amax((-1, -2))))
        x = _e4m3(x / scale[a:b, :, :, None, None])
        data[a:b] = x
        key = x[:, :, 0].float() / 4
        bounds[a:b, :, 0] = key.amin(-2).floor().to(torch.int8)
        bounds[a:b, :, 1] = key.amax(-2).ceil().to(torch.int8)
    return dict(data=data, scale=scale, bounds=bounds)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=dict(case))
    state.update({"rotary": _prepare_rotary, "verify": _prepare_verify, "copy": _prepare_copy}
                 .get(case["op"], _prepare_pool)(case, gen))
    return state


def _axes_of_pairs(case):
    """The axis of every pair: runs of pairs, the first axis (time) the shortest."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    edge = [0] + [pairs * (2 * i + 1) // (2 * axes) for i in range(1, axes)] + [pairs]
    return np.repeat(np.arange(axes), np.diff(edge))


def _prepare_rotary(case, gen):
    dev, kind = "cuda", TYPES[case["type"]]
    seqs, heads, dim, block = case["seqs"], case["kv_heads"], case["dim"], case["block"]
    before = _spread(case["low"], case["high"], seqs)
    count = _new_tokens(case)
    after = before + count
    blocks, skip = -(-after // block), before // block      # only blocks that the new tokens reach
    width = int(max(1, blocks.max()))
    pages = int((blocks - skip).sum()) + 3
    order = torch.randperm(pages, generator=gen, device=dev)
    at = torch.arange(width, device=dev)
    first = torch.from_numpy(np.cumsum(blocks - skip) - blocks).to(dev)[:, None]
    blocks_dev, skip_dev = torch.from_numpy(blocks).to(dev)[:, None], torch.from_numpy(skip).to(dev)[:, None]
    table = torch.where((at >= skip_dev) & (at < blocks_dev), order[(first + at).clamp(0, pages - 1)], -1)
    total = int(count.sum())
    # queries, keys and values are slices of one projection's output
    rows = case["q_heads"] + 2 * heads
    qkv = (1.5 * torch.randn((total, rows, dim), generator=gen, device=dev)).to(kind)
    # positions: runs of text, where the axes agree, and of images of 24 x 32 patches at one time
    token = torch.arange(total, device=dev)
    seq = torch.repeat_interleave(torch.arange(seqs, device=dev), torch.from_numpy(count).to(dev), output_size=total)
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(count)])).to(dev)
    place = token - offsets[seq] + torch.from_numpy(before).to(dev)[seq]
    image = (place // 768) % 3 == 1
    inside = place % 768
    by = [torch.where(image, place - inside, place), torch.where(image, place - inside + inside // 32, place),
          torch.where(image, place - inside + inside % 32, place), place // 2]
    pairs = case["rotated"] // 2
    freq = 1e6 ** (-torch.arange(pairs, dtype=torch.float64, device=dev) / pairs)
    return dict(_cache(gen, pages, heads, block, dim), table=table.to(torch.int32),
                q=qkv[:, :case["q_heads"]], k=qkv[:, case["q_heads"]:case["q_heads"] + heads],
                v=qkv[:, case["q_heads"] + heads:], start=torch.from_numpy(before).to(dev, torch.int32),
                offsets=offsets.to(torch.int32),
                positions=torch.stack(by[:case["axes"]]).to(torch.int32), freq=freq,
                axis=torch.from_numpy(_axes_of_pairs(case)).to(dev, torch.uint8),
                # how many blocks the tokens fall into: a program knows it from its own bookkeeping
                touched=int(np.where(count > 0, (after - 1) // block - before // block + 1, 0).sum()))


def _prepare_verify(case, gen):
    dev, kind = "cuda", TYPES[case["type"]]
    seqs, n, vocab = case["seqs"], case["tokens"], case["vocab"]
    logits = 2.5 * torch.randn((seqs, n + 1, vocab), generator=gen, device=dev)
    target = torch.softmax(logits, -1)
    if case["draft"]:
        # a smaller model that mostly agrees; tokens drawn from what it says
        logits = logits[:, :n] + 0.7 * torch.randn((seqs, n, vocab), generator=gen, device=dev)
        draft = torch.softmax(logits, -1).to(kind)
        source = draft.float()
    else:
        draft, source = None, target[:, :n]
    del logits
    edge = torch.rand((seqs, n, 1), generator=gen, device=dev, dtype=torch.float64)
    sums = source.double().cumsum(-1)
    tokens = torch.searchsorted(sums, edge * sums[..., -1:]).squeeze(-1).clamp(max=vocab - 1).to(torch.int32)
    accept = torch.rand((seqs, n), generator=gen, device=dev)
    if draft is None:
        accept *= accept * 0.01                 # one token of many: most random numbers reject it
    # tokens of a row are the newest of its sequence; a few rows have fewer drafts than others
    counts = torch.full((seqs,), n, dtype=torch.int32, device=dev)
    counts[4::5] -= 1
    return dict(target=target.to(kind), draft=draft, tokens=tokens, accept=accept,
                sample=torch.rand(seqs, generator=gen, device=dev), counts=counts,
                lengths=torch.randint(200, 30000, (seqs,), generator=gen, device=dev).to(torch.int32))


def _prepare_copy(case, gen):
    # from anywhere to anywhere, never to a page that is read
    order = torch.randperm(case["pages"], generator=gen, device="cuda").to(torch.int32)
    moves = case["moves"]
    return dict(_cache(gen, case["pages"], case["kv_heads"], case["block"], case["dim"]),
                src=order[:moves].contiguous(), dst=order[moves:2 * moves].contiguous())


def _prepare_pool(case, gen):
    dev, block, seqs, beams = "cuda", case["block"], case["seqs"], case.get("beams", 1)
    held = _lengths(case)
    want, evicted = held, 0
    if case["op"] == "resize":
        held, want = _wanted(case)
        evicted = case["evicted"]
    blocks = -(-held // block)
    goal = -(-want // block)
    width = int(max(1, blocks.max(), goal.max()))
    # every row has pages of its own, then beams take what they share from their first row
    own_pages = int(blocks.sum()) + evicted * seqs
    more = int(np.maximum(goal - blocks, 0).sum())
    pages = own_pages + 3 + int(case.get("spare", 0.0) * (own_pages + more)) + (more if case.get("spare") else more // 2)
    if case["op"] == "compact":
        pages = int(own_pages * 1.02) + 3
    order = torch.randperm(pages, generator=gen, device=dev)
    at = torch.arange(width, device=dev)
    row = torch.arange(seqs, device=dev)
    blocks_dev = torch.from_numpy(blocks).to(dev)[:, None]
    first = torch.from_numpy(np.cumsum(blocks) - blocks).to(dev)[:, None]
    index = first + at
    if beams > 1:
        lead = row - row % beams
        # half of the requests were forked just now, the others a while ago
        common = torch.where((row // beams) % 2 == 0, blocks_dev[:, 0], blocks_dev[:, 0] * 3 // 4)[:, None]
        index = torch.where(at < common, first[lead] + at, index)
    table = torch.where(at < blocks_dev, order[index.clamp(0, pages - 1)], -1).to(torch.int32)
    refs = _count(table, pages)
    state = dict(table=table, lengths=torch.from_numpy(held).to(dev, torch.int32))
    if case["op"] == "compact":
        # sequences that are gone: their rows are empty and their pages free
        away = torch.rand(seqs, generator=gen, device=dev) < case["gone"]
        state["table"] = table = torch.where(away[:, None], -1, table)
        refs = _count(table, pages)
    if case["op"] == "resize":
        state["want"] = torch.from_numpy(want).to(dev, torch.int32)
        if evicted:
            # pages that an eviction took out of the tables in the step before
            freed = torch.full((seqs, width), -1, dtype=torch.int32, device=dev)
            many = min(evicted, width)
            freed[:, :many] = order[own_pages - evicted * seqs + torch.arange(many * seqs, device=dev)].view(seqs, many).to(torch.int32)
            counts = ((row % (many + 1))).to(torch.int32)
            refs += _count(torch.where(at < counts[:, None], freed, -1), pages)
            state.update(freed=freed, freed_counts=counts)
    if case["op"] == "fork":
        # beams go on from any of their request's; a plain fork answers each row in turn
        rows = torch.arange(case["rows"], device=dev)
        if beams > 1:
            pick = torch.randint(0, beams, (case["rows"],), generator=gen, device=dev)
            parents = (rows % seqs) - (rows % seqs) % beams + pick
            parents = torch.where(torch.rand(case["rows"], generator=gen, device=dev) < 0.5, rows % seqs, parents)
        else:
            parents = rows * seqs // case["rows"]
        state["parents"] = torch.where(parents < seqs, parents, -1).to(torch.int32)
    return state | dict(refs=refs.to(torch.int32))


# ---------------------------------------------------------------------------
# One pass


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _rotary(s):
    c = s["case"]
    block, rotated, pairs = c["block"], c["rotated"], c["rotated"] // 2
    # angles, sines and cosines in 64 bits: positions are far, and stored values lie next to borders
    angle = (s["positions"].double()[s["axis"].long()].t() * s["freq"])[:, None]     # [tokens, 1, pairs]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def rotate(x):
        x = x.float()
        if c["neighbours"]:
            a, b = x[..., 0:rotated:2], x[..., 1:rotated:2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = x[..., :pairs], x[..., pairs:rotated]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([turned, x[..., rotated:]], -1)

    q, k = rotate(s["q"]).to(s["q"].dtype), rotate(s["k"])
    # the keys and values into the blocks of their sequences
    data, scale, bounds, table = s["data"], s["scale"], s["bounds"], s["table"]
    start, offsets = s["start"].long(), s["offsets"].long()
    count = offsets[1:] - offsets[:-1]
    first = start // block
    many = torch.where(count > 0, (start + count - 1) // block - first + 1, 0)
    seq = torch.repeat_interleave(torch.arange(many.numel(), device=many.device), many, output_size=s["touched"])
    index = torch.arange(s["touched"], device=many.device) - (many.cumsum(0) - many)[seq] + first[seq]
    page = table[seq, index].long()
    position = index[:, None] * block + torch.arange(block, device=many.device)
    old = position < start[seq, None]
    new = ~old & (position < (start + count)[seq, None])
    token = (offsets[seq, None] + position - start[seq, None]).clamp(0, k.shape[0] - 1)
    fresh = torch.stack([k[token], s["v"][token].float()], 1).permute(0, 3, 1, 2, 4)
    old, new = old[:, None, None, :, None], new[:, None, None, :, None]
    need = _power(_exponent(torch.where(new & fresh.isfinite(), fresh.abs(), 0).amax((-1, -2))))
    was = scale[page]
    now = torch.where(old.any(-2).squeeze(-1), torch.maximum(was, need), need)
    held = data.view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * (was / now)[..., None, None]
    values = _e4m3(torch.where(new, fresh / now[..., None, None], torch.where(old, held, 0)))
    data.view(torch.uint8)[page] = values.view(torch.uint8)
    scale[page] = now
    key = values[:, :, 0].float().nan_to_num() / 4
    used = (old | new)[:, :, 0]
    bounds[page] = torch.stack([torch.where(used, key, math.inf).amin(-2).floor(),
                                torch.where(used, key, -math.inf).amax(-2).ceil()], 2).to(torch.int8)
    return {"q": q, "data": data, "scale": scale, "bounds": bounds}


def _whole(p):
    """Probabilities as whole multiples of 2^-40; exact in 64 bits, halves to even."""
    return (p.double().nan_to_num(nan=0.0).clamp(0, 1) * 2.0 ** 40).round().to(torch.int64)


def _verify(s):
    target, draft, tokens = s["target"], s["draft"], s["tokens"]
    seqs, n, dev = tokens.shape[0], tokens.shape[1], tokens.device
    vocab = target.shape[-1]
    at = torch.arange(n, device=dev)
    real = (tokens >= 0) & (tokens < vocab) & (at < s["counts"][:, None])
    index = torch.where(real, tokens, 0).long()[..., None]
    p = target[:, :n].gather(2, index).squeeze(2).double()
    q = draft.gather(2, index).squeeze(2).double() if draft is not None else torch.ones_like(p)
    good = real & (s["accept"].double() * q < p)        # products of 24 bits each are exact
    accepted = good.long().cumprod(1).sum(1)
    row = torch.arange(seqs, device=dev)
    left = _whole(target[row, accepted])
    spare = left
    inside = (accepted < s["counts"])[:, None]
    if draft is not None:
        away = _whole(draft[row, accepted.clamp(max=n - 1)])
    else:
        chosen = index.squeeze(2).gather(1, accepted.clamp(max=n - 1)[:, None])
        known = real.gather(1, accepted.clamp(max=n - 1)[:, None])
        away = torch.where((torch.arange(vocab, device=dev) == chosen) & known, left, 0)
    left = torch.where(inside, (left - away).clamp(min=0), left)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, spare)
    sums = left.cumsum(1)
    total = sums[:, -1:]
    u = (s["sample"].double().nan_to_num(nan=0.0) * 2 ** 24).floor().clamp(0, 2 ** 24 - 1).to(torch.int64)[:, None]
    # floor(u * total / 2^24) in parts that fit 64 bits
    border = (u * (total >> 32) << 8) + (u * (total & 0xffffffff) >> 24)
    picked = (sums <= border).sum(1)
    picked = torch.where(total.squeeze(1) > 0, picked, -1)
    out = torch.where(at < accepted[:, None], tokens, -1)
    out = torch.cat([out, out.new_full((seqs, 1), -1)], 1)
    out = out.scatter(1, accepted[:, None], picked[:, None].to(out.dtype))
    lengths = s["lengths"] - (s["counts"] - accepted)
    return {"accepted": accepted.to(torch.int32), "tokens": out, "lengths": lengths.to(torch.int32)}


def _count(table, pages):
    """How often each page is named."""
    named = torch.where((table >= 0) & (table < pages), table, pages).long().flatten()
    return torch.zeros(pages + 1, dtype=torch.int64, device=table.device).scatter_add_(
        0, named, torch.ones_like(named))[:pages]


def _resize(s):
    block, table, dev = s["case"]["block"], s["table"], s["table"].device
    pages, (seqs, width) = s["refs"].numel(), table.shape
    held, goal = (x.long().clamp(0, width * block) for x in (s["lengths"], s["want"]))
    need = (goal + block - 1) // block
    at, row = torch.arange(width, device=dev), torch.arange(seqs, device=dev)[:, None]
    behind = at >= need[:, None]
    # pages behind the rows' new ends and evicted ones go back
    refs = s["refs"].long() - _count(torch.where(behind, table, -1), pages)
    if "freed" in s:
        listed_now = torch.arange(s["freed"].shape[1], device=dev) < s["freed_counts"][:, None]
        refs = refs - _count(torch.where(listed_now, s["freed"], -1), pages)
    table = torch.where(behind, -1, table)
    # blocks that new tokens reach: without a page, or with one that others name too
    asked = (at >= (held // block)[:, None]) & ~behind & (goal > held)[:, None]
    there = (table >= 0) & (table < pages)
    page = torch.where(there, table, 0).long()
    shared = asked & there & (refs[page] > 1)
    named = torch.where(shared, page, pages)
    claims = torch.zeros(pages + 1, dtype=torch.int64, device=dev).scatter_add_(
        0, named.flatten(), torch.ones_like(named).flatten())
    last = torch.full((pages + 1,), -1, dtype=torch.int64, device=dev).scatter_reduce_(
        0, named.flatten(), row.expand(seqs, width).flatten(), "amax")
    stays = shared & (claims[page] >= refs[page]) & (last[page] == row)
    claim = (asked & ~there) | (shared & ~stays)
    before = claim.flatten().cumsum(0).view(seqs, width) - claim.long()
    # free pages, the lowest first
    free = refs <= 0
    rank = torch.where(free, free.cumsum(0) - 1, pages)
    pool = torch.zeros(pages + 1, dtype=torch.int64, device=dev).scatter_(0, rank, torch.arange(pages, device=dev))
    many = free.sum()
    served = claim & (before < many)
    given = pool[torch.where(served, before, pages)]
    parted = served & shared
    refs = refs - _count(torch.where(parted, page, -1), pages)
    mark = torch.cat([refs, refs.new_zeros(1)]).scatter_(0, torch.where(served, given, pages).flatten(),
                                                         torch.ones_like(given).flatten())
    new_table = torch.where(served, given, table.long()).to(torch.int32)
    # contents that have to follow: the block that new tokens go on in
    part = parted & (at == (held // block)[:, None]) & (held % block != 0)[:, None]
    src = torch.where(part, page, -1).amax(1)
    dst = torch.where(part, given, -1).amax(1)
    stuck = (claim & ~served) | (stays & (before > many))
    stop = torch.where(stuck, at, width).amin(1)
    limits = torch.where(stuck.any(1), torch.maximum(held, stop * block), goal)
    return {"refs": mark[:pages].to(torch.int32), "table": new_table, "limits": limits.to(torch.int32),
            "src": src.to(torch.int32), "dst": dst.to(torch.int32)}


def _fork(s):
    block, table, parents = s["case"]["block"], s["table"], s["parents"].long()
    seqs, width = table.shape
    real = (parents >= 0) & (parents < seqs)
    parent = torch.where(real, parents, 0)
    held = s["lengths"].long().clamp(0, width * block)[parent]
    keep = real[:, None] & (torch.arange(width, device=table.device) < ((held + block - 1) // block)[:, None])
    new = torch.where(keep, table[parent], -1)
    pages = s["refs"].numel()
    refs = s["refs"].long() + _count(new, pages) - _count(table, pages)
    return {"refs": refs.to(torch.int32), "table": new, "lengths": torch.where(real, held, 0).to(torch.int32)}


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    data = s["data"].view(torch.uint8)
    data[dst] = data[src]
    s["scale"][dst] = s["scale"][src]
    s["bounds"][dst] = s["bounds"][src]
    return {"data": s["data"], "scale": s["scale"], "bounds": s["bounds"]}


def _compact(s):
    refs, table, dev = s["refs"], s["table"], s["table"].device
    pages = refs.numel()
    at = torch.arange(pages, device=dev)
    live = refs > 0
    below = live.cumsum(0)
    many = below[-1]
    room = pages // 2
    moves = torch.full((2, room + 1), -1, dtype=torch.int64, device=dev)
    # the highest page in use goes to the lowest free page, the next to the next
    from_top = torch.where(live & (at >= many), many - below, room)
    from_bottom = torch.where(~live & (at < many), at - below, room)
    moves[0].scatter_(0, from_top, at)
    moves[1].scatter_(0, from_bottom, at)
    moves[:, room] = -1
    src, dst = moves[0], moves[1]
    where = torch.where(live, at, -1)
    there = (src >= 0)
    where = torch.cat([where, where.new_zeros(1)]).scatter_(0, torch.where(there, src, pages), dst)[:pages]
    new_refs = torch.cat([torch.where(live, refs, 0), refs.new_zeros(1)])
    new_refs = new_refs.scatter(0, torch.where(there, dst, pages), new_refs[torch.where(there, src, pages)])[:pages]
    new_refs = torch.where(at < many, new_refs, 0)
    named = (table >= 0) & (table < pages)
    new_table = torch.where(named, where[torch.where(named, table, 0).long()], table.long())
    return {"refs": new_refs.to(torch.int32), "table": new_table.to(torch.int32), "src": src[:room].to(torch.int32),
            "dst": dst[:room].to(torch.int32), "live": many.view(1).to(torch.int32), "where": where.to(torch.int32)}


_plain = {"rotary": _rotary, "verify": _verify, "resize": _resize, "fork": _fork, "copy": _copy,
          "compact": _compact}


def _own_rotary(s):
    import hbfsim_b200 as hbf
    rotary = hbf.KvRotary(s["freq"], s["axis"], neighbours=s["case"]["neighbours"])
    q = hbf.kv_append_rotary(hbf.KvCache(s["data"], s["scale"], s["bounds"]), s["q"], s["k"], s["v"],
                             s["table"], s["start"], s["positions"], rotary, offsets=s["offsets"])
    return {"q": q, "data": s["data"], "scale": s["scale"], "bounds": s["bounds"]}


def _own_verify(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_verify(s["target"], s["draft"], s["tokens"], s["accept"], s["sample"],
                        counts=s["counts"], lengths=s["lengths"])
    return {"accepted": got.accepted, "tokens": got.tokens, "lengths": got.lengths}


def _own_resize(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_resize(s["refs"], s["table"], s["lengths"], s["want"], block_tokens=s["case"]["block"],
                        freed=s.get("freed"), freed_counts=s.get("freed_counts"))
    return {"refs": got.refs, "table": got.table, "limits": got.limits, "src": got.src, "dst": got.dst}


def _own_fork(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_fork(s["refs"], s["table"], s["lengths"], s["parents"], block_tokens=s["case"]["block"])
    return {"refs": got.refs, "table": got.table, "lengths": got.lengths}


def _own_copy(s):
    import hbfsim_b200 as hbf
    hbf.kv_copy(hbf.KvCache(s["data"], s["scale"], s["bounds"]), s["src"], s["dst"])
    return {"data": s["data"], "scale": s["scale"], "bounds": s["bounds"]}


def _own_compact(s):
    import hbfsim_b200 as hbf
    got = hbf.kv_compact(s["refs"], s["table"])
    return {"refs": got.refs, "table": got.table, "src": got.src, "dst": got.dst, "live": got.live,
            "where": got.where}


_own = {"rotary": _own_rotary, "verify": _own_verify, "resize": _own_resize, "fork": _own_fork,
        "copy": _own_copy, "compact": _own_compact}


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    op = case["op"]
    if op == "rotary":
        heads, dim, block = case["kv_heads"], case["dim"], case["block"]
        before, count = _spread(case["low"], case["high"], case["seqs"]), _new_tokens(case)
        total = int(count.sum())
        touched = int(np.where(count > 0, (before + count - 1) // block - before // block + 1, 0).sum())
        # queries in and out; keys and values in, their 8-bit forms out; scales and bounds
        return {"bytes": total * (case["q_heads"] * dim * 4 + heads * dim * 2 * 3 + 4 * case["axes"])
                + touched * heads * (8 + 2 * dim),
                "flops": total * (3 * case["rotated"] * (case["q_heads"] + heads) + 4 * heads * dim * 2)}
    if op == "verify":
        # the row that the next token comes from, and the draft's where one was rejected (here: counted
        # for every sequence, most of which have one)
        values = case["seqs"] * case["vocab"] * (2 if case["draft"] else 1)
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": values * size + case["seqs"] * case["tokens"] * 16, "flops": 3 * values}
    if op == "copy":
        page = case["kv_heads"] * (2 * case["block"] * case["dim"] + 2 * case["dim"] + 8)
        return {"bytes": case["moves"] * (2 * page + 8), "flops": case["moves"]}
    seqs, block = case["seqs"], case["block"]
    if op == "resize":
        held, want = _wanted(case)
    else:
        held = want = _lengths(case)
    blocks, goal = -(-held // block), -(-want // block)
    width = int(max(1, blocks.max(), goal.max()))
    own_pages = int(blocks.sum())
    if op == "fork":
        # the parents' rows in, the children's out, counts in and out
        return {"bytes": 4 * own_pages + 4 * case["rows"] * width + 8 * own_pages, "flops": case["rows"] * width}
    if op == "compact":
        # counts in and out, the new place of every page, the table in and out
        return {"bytes": 12 * own_pages + 8 * seqs * width, "flops": own_pages + seqs * width}
    more = int(np.maximum(goal - blocks, 0).sum())
    return {"bytes": 8 * (own_pages + more) + 8 * seqs * width, "flops": own_pages + more + seqs * width}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _round_e4m3(x):
    """Nearest value of 4 significant bits (ties to even), steps of 2^-9 below 2^-6, at most 448."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    step = torch.where(size / step >= 16, step * 2, torch.where(size / step < 8, step / 2, step))
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_rotary(s):
    case = s["case"]
    block, pairs = case["block"], case["rotated"] // 2
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    for i in range(pairs):
        a = (s["positions"][int(s["axis"][i])].double() * s["freq"][i])[:, None]
        c0, c1 = (2 * i, 2 * i + 1) if case["neighbours"] else (i, i + pairs)
        for x in (q, k):
            first, second = x[..., c0].clone(), x[..., c1].clone()
            x[..., c0] = torch.cos(a) * first - torch.sin(a) * second
            x[..., c1] = torch.sin(a) * first + torch.cos(a) * second
    start, offsets, table = s["start"].tolist(), s["offsets"].tolist(), s["table"].tolist()
    data, scale = s["data"].double(), s["scale"].double()
    for b in range(case["seqs"]):
        done, count = 0, offsets[b + 1] - offsets[b]
        while done < count:
            p = start[b] + done
            page, slot = table[b][p // block], p % block
            many = min(block - slot, count - done)
            x = torch.stack([k[offsets[b] + done:][:many], v[offsets[b] + done:][:many]]).permute(2, 0, 1, 3)
            size = x.abs().amax((2, 3))                                 # [heads, 2]
            need = torch.exp2(torch.ceil(torch.log2(size / 448.0)).clamp(LOWEST, HIGHEST))
            need = torch.where(size > 448.0 * need, 2 * need, need)
            need = torch.where((size <= 224.0 * need) & (need > 2.0 ** LOWEST), need / 2, need)
            now = torch.maximum(need, scale[page]) if slot else need
            data[page, :, :, :slot] = _round_e4m3(data[page, :, :, :slot] * (scale[page] / now)[..., None, None])
            data[page, :, :, slot:] = 0
            data[page, :, :, slot:slot + many] = _round_e4m3(x / now[..., None, None])
            scale[page] = now
            done += many
    return {"q": q, "data": data, "scale": scale, "bounds": None}


def _exact_copy(s):
    source = np.arange(s["case"]["pages"])
    source[s["dst"].cpu().numpy()] = s["src"].cpu().numpy()
    source = torch.from_numpy(source).cuda()
    return {"data": s["data"].view(torch.uint8)[source].view(torch.float8_e4m3fn).double(),
            "scale": s["scale"].double()[source], "bounds": None}


def exact(case, seed):
    if case["op"] == "copy":
        return _exact_copy(prepare(case, seed))
    if case["op"] != "rotary":
        return None                     # whole numbers, which the plain form gives exactly
    if case["seqs"] * max(1, case["tokens"] // case["block"]) > 4000:
        return None                     # one block at a time: too many of them
    return _exact_rotary(prepare(case, seed))
