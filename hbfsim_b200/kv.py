"""Operators over a paged key/value cache held in 8 bits (include/hbfsim/kv_v1.h).

One decode step of a layer is

    kv_append(cache, k, v, table, start)                 # the new tokens' keys and values
    pick = kv_select(cache, q, table, lengths, top=128)  # blocks worth reading, per head
    got = kv_attention(cache, q, table, lengths, blocks=pick.blocks,
                       counts=pick.counts, weights=True)
    rest = kv_evict(score, got.weights, table, lengths, keep=...)
    reads = kv_block_reads(cache, table, pick.blocks, pick.counts, base)  # for Context.submit

kv_attention without lists reads every block.  Around it:

    room = kv_resize(refs, table, lengths, want)         # pages for the step's tokens, or back
    kv_copy(cache, room.src, room.dst)                   # blocks that were shared, every layer
    q = kv_append_rotary(cache, q, k, v, table, start, positions, rotary)  # positions turned in
    kept = kv_verify(target, draft, tokens, accept, sample, lengths=lengths)  # drafted tokens
    kv_fork, kv_compact                                  # children of sequences; a smaller pool

Arguments that do not fit raise ValueError here, or HbfsimError from the C ABI; so do keys, values and
queries that ask for a gradient, since there is no backward pass (inside
torch.no_grad() they are taken as they are).  Calls are asynchronous
on `stream` (default: torch's current stream); outputs and workspace belong
to that stream.
"""
from __future__ import annotations

import struct
from typing import NamedTuple

from . import _lib
from ._lib import check
from .api import CUDA_STREAM_LEGACY

__all__ = ["KvCache", "KvAttention", "KvSelection", "KvEviction", "KvRotary", "KvVerified",
           "KvResized", "KvForked", "KvCompacted", "kv_append", "kv_append_rotary", "kv_attention",
           "kv_select", "kv_evict", "kv_block_reads", "kv_verify", "kv_resize", "kv_fork",
           "kv_copy", "kv_compact"]

# The C structures of kv_v1.h as packed bytes (no padding: 8-byte fields lie at multiples of 8);
# _lib has the same structures field by field.
_CACHE = struct.Struct("<6I4Q")
_APPEND = struct.Struct("<6I3Q4qQq2Q")
_QUERY = struct.Struct("<8IQ3qQqQ")
_ATTENTION = struct.Struct("<2IfI7Q")
_EVICT = struct.Struct("<10I3Qq6Q")
_ROTARY = struct.Struct("<6IQ2q2Qq2Q")
_VERIFY = struct.Struct("<6IQ2qQ2q8Q")
_RESIZE = struct.Struct("<8I3Qq6Qq3Q")  # both without their workspace
_FORK = struct.Struct("<6I3Qq5Q")
_COMPACT = struct.Struct("<4I3Qq2Qq4Q")
_WORKSPACE = struct.Struct("<2Q")
_NO_WORKSPACE = _WORKSPACE.pack(0, 0)


_NO_GRADIENT = "no gradient passes through the cache: detach the tensors or call under torch.no_grad()"


class KvAttention(NamedTuple):
    out: object
    lse: object
    weights: object


class KvSelection(NamedTuple):
    blocks: object
    counts: object


class KvEviction(NamedTuple):
    score: object
    table: object
    lengths: object
    freed: object
    freed_counts: object


class KvVerified(NamedTuple):
    accepted: object
    tokens: object
    lengths: object


class KvResized(NamedTuple):
    refs: object
    table: object
    limits: object
    src: object
    dst: object


class KvForked(NamedTuple):
    refs: object
    table: object
    lengths: object


class KvCompacted(NamedTuple):
    refs: object
    table: object
    src: object
    dst: object
    live: object
    where: object


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class KvCache:
    """The cache's three tensors (a view of them; nothing is copied):
    data (float8_e4m3fn [pages, kv_heads, 2, block_tokens, head_dim]), scale
    (float32 [pages, kv_heads, 2]), bounds (int8 [pages, kv_heads, 2,
    head_dim]).  The layout and the meaning are in kv_v1.h."""

    __slots__ = ("data", "scale", "bounds", "pages", "kv_heads", "block_tokens", "head_dim",
                 "index", "_packed")

    def __init__(self, data, scale, bounds):
        import torch
        shape = data.shape
        _need(len(shape) == 5 and shape[2] == 2 and data.dtype == torch.float8_e4m3fn,
              "data: float8_e4m3fn [pages, kv_heads, 2, block_tokens, head_dim]")
        pages, heads, _, block, dim = shape
        _need(scale.dtype == torch.float32 and scale.shape == (pages, heads, 2),
              "scale: float32 [pages, kv_heads, 2]")
        _need(bounds.dtype == torch.int8 and bounds.shape == (pages, heads, 2, dim),
              "bounds: int8 [pages, kv_heads, 2, head_dim]")
        _need(data.is_contiguous() and scale.is_contiguous() and bounds.is_contiguous(),
              "data, scale and bounds have to be contiguous")
        self.index = index = data.get_device()  # of the CUDA device
        _need(index >= 0 and scale.get_device() == index and bounds.get_device() == index,
              "data, scale and bounds have to be on one CUDA device")
        self.data, self.scale, self.bounds = data, scale, bounds
        self.pages, self.kv_heads, self.block_tokens, self.head_dim = pages, heads, block, dim
        self._packed = _CACHE.pack(_CACHE.size, 1, heads, dim, block, 0, pages, data.data_ptr(),
                                   scale.data_ptr(), bounds.data_ptr())

    @property
    def device(self):
        return self.data.device

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int = 128, block_tokens: int = 16,
              device="cuda") -> "KvCache":
        """A cache of `pages` pages of zeros."""
        import torch
        data = torch.zeros((pages, kv_heads, 2, block_tokens, head_dim), dtype=torch.uint8,
                           device=device).view(torch.float8_e4m3fn)
        scale = torch.ones((pages, kv_heads, 2), dtype=torch.float32, device=device)
        bounds = torch.zeros((pages, kv_heads, 2, head_dim), dtype=torch.int8, device=device)
        return cls(data, scale, bounds)

    @property
    def block_bytes(self) -> int:
        """Bytes of one head's keys and values of a block."""
        return 2 * self.block_tokens * self.head_dim


def _type(t) -> int:
    import torch
    if t.dtype == torch.bfloat16:
        return _lib.KV_BF16
    _need(t.dtype == torch.float16, "keys, values and queries are bfloat16 or float16")
    return _lib.KV_F16


def _check_table(index, table, per_seq, name):
    """Shape of the block table; `per_seq` is the int32 tensor that goes with its rows."""
    import torch
    shape = table.shape
    _need(len(shape) == 2 and table.dtype == torch.int32 and table.get_device() == index
          and (table.stride(1) == 1 or shape[1] <= 1 or shape[0] == 0),
          "table: int32 [seqs, width] on the cache's device, rows contiguous")
    _need(per_seq.dtype == torch.int32 and per_seq.shape == shape[:1]
          and per_seq.get_device() == index and (per_seq.stride(0) == 1 or shape[0] <= 1),
          f"{name}: int32 [seqs] on the cache's device, contiguous")
    return shape


class _On:
    """Makes a device and a stream current for the allocations of a call."""

    def __init__(self, index, stream):
        import torch
        _need(stream is None or stream.device.index == index, "the stream is of another device")
        self.inside = [torch.cuda.device(index)]
        if stream is not None:
            self.inside.append(torch.cuda.stream(stream))

    def __enter__(self):
        for x in self.inside:
            x.__enter__()

    def __exit__(self, *exc):
        for x in reversed(self.inside):
            x.__exit__(*exc)


def _here(index, stream) -> bool:
    """Whether the call's device is current and its stream is the current one."""
    import torch
    return stream is None and torch._C._cuda_getDevice() == index


def _handle(index) -> int:
    import torch
    return torch._C._cuda_getCurrentRawStream(index) or CUDA_STREAM_LEGACY


def kv_append(cache: KvCache, k, v, table, start, offsets=None, stream=None) -> None:
    """Quantises new tokens into the blocks of their sequences.

    k, v: [seqs, n, kv_heads, head_dim], or with `offsets` (int32 [seqs + 1])
    ragged [tokens, kv_heads, head_dim], sequence s owning tokens
    [offsets[s], offsets[s + 1]); any strides with a contiguous last axis.
    start: int32 [seqs], tokens a sequence held before.  Writes data, scale
    and bounds of the touched blocks in place."""
    if not _here(cache.index, stream):
        with _On(cache.index, stream):
            return kv_append(cache, k, v, table, start, offsets)
    batch, tokens, _held = _append(cache, k, v, table, start, offsets)
    if tokens:
        check(_lib.load().hbfsim_kv_append_v1(cache._packed, batch, _handle(cache.index)),
              "hbfsim_kv_append_v1")


def _append(cache: KvCache, k, v, table, start, offsets) -> tuple:
    """The packed append, its tokens, and what has to live until the launch (copies of k and v)."""
    import torch
    seqs, width = _check_table(cache.index, table, start, "start")
    shape = k.shape
    _need(shape == v.shape and k.dtype == v.dtype and k.get_device() == cache.index
          and v.get_device() == cache.index and len(shape) == (4 if offsets is None else 3)
          and shape[-2] == cache.kv_heads and shape[-1] == cache.head_dim,
          "k and v: one shape and type, [seqs, n, kv_heads, head_dim] or with offsets "
          "[tokens, kv_heads, head_dim], on the cache's device")
    _need(not (k.requires_grad or v.requires_grad) or not torch.is_grad_enabled(), _NO_GRADIENT)
    if offsets is None:
        _need(shape[0] == seqs, "k: as many sequences as the table")
        k, v = k.flatten(0, 1), v.flatten(0, 1)  # a copy where one stride cannot serve both axes
        at = 0
    else:
        _need(offsets.dtype == torch.int32 and offsets.shape == (seqs + 1,)
              and offsets.get_device() == cache.index and offsets.is_contiguous(),
              "offsets: int32 [seqs + 1] on the cache's device, contiguous")
        at = offsets.data_ptr()
    tokens = k.shape[0]
    if tokens == 0:
        return b"", 0, None
    k_token, k_head, k_dim = k.stride()
    v_token, v_head, v_dim = v.stride()
    _need(k_dim == 1 and v_dim == 1, "the last axis of k and v has to be contiguous")
    return _APPEND.pack(_APPEND.size, 1, _type(k), seqs, width, 0, tokens, k.data_ptr(),
                        v.data_ptr(), k_token, k_head, v_token, v_head, table.data_ptr(),
                        table.stride(0), start.data_ptr(), at), tokens, (k, v)


class KvRotary:
    """How pairs of channels turn with their positions (a view of two tensors):
    freq (float64 [pairs], radians a position) and axis (uint8 [pairs], which
    axis of the positions a pair follows).  A head's first 2 * pairs channels are
    turned: channel i with i + pairs, or with `neighbours` 2i with 2i + 1."""

    __slots__ = ("freq", "axis", "pairs", "neighbours", "index")

    def __init__(self, freq, axis, neighbours: bool = False):
        import torch
        _need(freq.dtype == torch.float64 and freq.dim() == 1 and freq.is_contiguous(),
              "freq: float64 [pairs], contiguous")
        _need(axis.dtype == torch.uint8 and axis.shape == freq.shape and axis.is_contiguous(),
              "axis: uint8 [pairs], contiguous")
        self.index = index = freq.get_device()
        _need(index >= 0 and axis.get_device() == index,
              "freq and axis have to be on one CUDA device")
        self.freq, self.axis, self.neighbours = freq, axis, bool(neighbours)
        self.pairs = freq.shape[0]

    @classmethod
    def of(cls, head_dim: int, base: float = 10000.0, rotated: int | None = None, sections=None,
           neighbours: bool = False, device="cuda") -> "KvRotary":
        """Frequencies base ** (-2 i / rotated) for the first `rotated` channels (default: all);
        `sections`: how many pairs in turn follow each axis (default: all the only one)."""
        import torch
        rotated = head_dim if rotated is None else rotated
        _need(0 < rotated <= head_dim and rotated % 2 == 0, "rotated: an even number of channels")
        pairs = rotated // 2
        sections = (pairs,) if sections is None else tuple(sections)
        _need(1 <= len(sections) <= 4 and min(sections) >= 0 and sum(sections) == pairs,
              "sections: one to four numbers of pairs that add up to rotated / 2")
        freq = float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
        axis = torch.repeat_interleave(torch.arange(len(sections), dtype=torch.uint8),
                                       torch.tensor(sections))
        return cls(freq.to(device), axis.to(device), neighbours)


def kv_append_rotary(cache: KvCache, q, k, v, table, start, positions, rotary: KvRotary,
                     offsets=None, stream=None):
    """kv_append with the keys turned by their positions on the way into the cache, and the queries
    of the same tokens with them.

    k, v, table, start, offsets: as for kv_append.  q: [seqs, n, q_heads, head_dim], or with
    `offsets` [tokens, q_heads, head_dim], of k's type; None: keys alone.  positions: int32 [axes,
    seqs, n], or with `offsets` [axes, tokens], 1 to 4 axes (a single one may be left out).
    rotary: a KvRotary on the cache's device; its pairs are a multiple of head_dim / 32.

    Returns the turned queries (q's type and shape; every row, rows that belong to no sequence
    too), None without q."""
    if not _here(cache.index, stream):
        with _On(cache.index, stream):
            return kv_append_rotary(cache, q, k, v, table, start, positions, rotary, offsets)
    import torch
    batch, tokens, _held = _append(cache, k, v, table, start, offsets)
    lead = k.shape[:-2]
    _need(rotary.index == cache.index, "rotary: on the cache's device")
    axes = positions.shape[0] if positions.dim() == len(lead) + 1 else 1
    _need(positions.dtype == torch.int32 and positions.get_device() == cache.index
          and positions.shape[-len(lead):] == lead and positions.dim() <= len(lead) + 1
          and 1 <= axes <= 4, "positions: int32 [axes, seqs, n] or with offsets [axes, tokens], 1 to 4 "
          "axes, on the cache's device")
    out, q_heads, q_at, q_token, q_head = None, 0, 0, 0, 0
    if q is not None:
        _need(q.dtype == k.dtype and q.get_device() == cache.index and q.dim() == len(lead) + 2
              and q.shape[:-2] == lead and q.shape[-1] == cache.head_dim,
              "q: [seqs, n, q_heads, head_dim] or with offsets [tokens, q_heads, head_dim], of k's "
              "type, on the cache's device")
        _need(not q.requires_grad or not torch.is_grad_enabled(), _NO_GRADIENT)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q_heads = q.shape[-2]
        if q_heads and tokens:
            if offsets is None:
                q = q.flatten(0, 1)
            q_token, q_head, q_dim = q.stride()
            _need(q_dim == 1, "the last axis of q has to be contiguous")
            q_at = q.data_ptr()
    if tokens == 0:
        return out
    places = positions if offsets is not None and positions.dim() == 2 else positions.reshape(axes, tokens)
    if places.stride(1) != 1 and tokens > 1:
        places = places.contiguous()
    packed = _ROTARY.pack(_ROTARY.size, 1, q_heads, axes, rotary.pairs, rotary.neighbours, q_at,
                          q_token, q_head, out.data_ptr() if q_heads else 0, places.data_ptr(),
                          places.stride(0), rotary.freq.data_ptr(), rotary.axis.data_ptr())
    check(_lib.load().hbfsim_kv_append_rotary_v1(cache._packed, batch, packed,
                                                 _handle(cache.index)),
          "hbfsim_kv_append_rotary_v1")
    return out


def _query(cache: KvCache, q, table, lengths) -> tuple:
    """The packed query and its sizes: (bytes, seqs, tokens, q_heads, width)."""
    table_seqs, width = _check_table(cache.index, table, lengths, "lengths")
    _need(q.dim() == 4 and q.get_device() == cache.index,
          "q: [seqs, tokens, q_heads, head_dim] on the cache's device")
    seqs, tokens, q_heads, dim = q.shape
    _need(seqs == table_seqs and dim == cache.head_dim,
          "q: [seqs, tokens, q_heads, head_dim] with the table's seqs and the cache's head_dim")
    _need(q_heads > 0 and q_heads % cache.kv_heads == 0, "q_heads has to be a multiple of kv_heads")
    by_seq, by_token, by_head, by_dim = q.stride()
    _need(by_dim == 1, "the last axis of q has to be contiguous")
    packed = _QUERY.pack(_QUERY.size, 1, _type(q), seqs, tokens, q_heads, width, 0, q.data_ptr(),
                         by_seq, by_token, by_head, table.data_ptr(), table.stride(0),
                         lengths.data_ptr())
    return packed, seqs, tokens, q_heads, width


def kv_select(cache: KvCache, q, table, lengths, top: int, sink: int = 1, recent: int = 1,
              stream=None) -> KvSelection:
    """For every query token and key/value head the blocks worth reading: the
    first `sink`, the last `recent` and those whose bounds allow the largest
    products with the group's queries, `top` in all.

    q: [seqs, tokens, q_heads, head_dim], the newest tokens, which `lengths`
    counts.  Returns blocks (int32 [seqs, tokens, kv_heads, top], ascending,
    -1 behind the count) and counts (int32 [seqs, tokens, kv_heads])."""
    if not _here(cache.index, stream):
        with _On(cache.index, stream):
            return kv_select(cache, q, table, lengths, top, sink, recent)
    _need(not (top | sink | recent) >> 32, "top, sink and recent are counts of 32 bits")
    _need(top <= 1 << 24, "a list has room for 2^24 blocks at most")  # as many as a table
    query, seqs, tokens, _, _ = _query(cache, q, table, lengths)
    lib = _lib.load()
    blocks = table.new_empty((seqs, tokens, cache.kv_heads, top))
    counts = table.new_empty((seqs, tokens, cache.kv_heads))
    size = lib.hbfsim_kv_select_workspace_v1(cache._packed, query)
    space = cache.bounds.new_empty(size)
    check(lib.hbfsim_kv_select_v1(cache._packed, query, top, sink, recent, blocks.data_ptr(),
                                  counts.data_ptr(), space.data_ptr(), size, _handle(cache.index)),
          "hbfsim_kv_select_v1")
    return KvSelection(blocks, counts)


def kv_attention(cache: KvCache, q, table, lengths, scale: float | None = None, blocks=None,
                 counts=None, weights: bool = False, stream=None) -> KvAttention:
    """Attention of the newest tokens: q [seqs, tokens, q_heads, head_dim],
    token t at position lengths - tokens + t.  scale: of the products
    (default head_dim ** -0.5).  blocks, counts: lists as kv_select returns
    them (default: every block).  The table's width decides how the call is
    spread over the device: narrow it (table[:, :n]) where all sequences are
    known to be short.

    Returns out (q's type and shape), lse (float32 [seqs, tokens, q_heads],
    natural logarithm of the sum of exponentials) and, if asked for, weights
    (float32 [seqs, kv_heads, width]: softmax weight of every block, summed
    over the group's heads and the tokens; else None)."""
    if not _here(cache.index, stream):
        with _On(cache.index, stream):
            return kv_attention(cache, q, table, lengths, scale, blocks, counts, weights)
    import torch
    _need(not q.requires_grad or not torch.is_grad_enabled(), _NO_GRADIENT)
    query, seqs, tokens, q_heads, width = _query(cache, q, table, lengths)
    top = blocks_at = counts_at = 0
    if blocks is not None:
        shape = (seqs, tokens, cache.kv_heads)
        _need(counts is not None and blocks.dtype == torch.int32 and counts.dtype == torch.int32
              and blocks.dim() == 4 and blocks.shape[:3] == shape and counts.shape == shape
              and blocks.is_contiguous() and counts.is_contiguous()
              and blocks.get_device() == cache.index and counts.get_device() == cache.index,
              "blocks and counts: int32 [seqs, tokens, kv_heads(, top)] on the cache's device, "
              "contiguous")
        top = blocks.shape[3]
        _need(top > 0, "a list has to have room for one block")
        blocks_at, counts_at = blocks.data_ptr() or 16, counts.data_ptr() or 16  # 0: no lists
    else:
        _need(counts is None, "counts without blocks")
    lib = _lib.load()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = cache.scale.new_empty((seqs, tokens, q_heads))
    mass, mass_at = None, 0
    if weights:
        # with no query token nothing is launched and every weight is 0
        make = cache.scale.new_empty if tokens else cache.scale.new_zeros
        mass = make((seqs, cache.kv_heads, width))
        mass_at = mass.data_ptr()
    if scale is None:
        scale = cache.head_dim ** -0.5
    else:
        _need(not abs(scale) > 3.0e38, "the scale has to fit 32 bits")
    head = (_ATTENTION.size, 1, scale, top, blocks_at, counts_at, out.data_ptr(), lse.data_ptr(),
            mass_at)
    size = lib.hbfsim_kv_attention_workspace_v1(cache._packed, query, _ATTENTION.pack(*head, 0, 0))
    space = cache.bounds.new_empty(size) if size else None  # held until the launch
    space_at = space.data_ptr() if size else 0
    check(lib.hbfsim_kv_attention_v1(cache._packed, query, _ATTENTION.pack(*head, space_at, size),
                                     _handle(cache.index)), "hbfsim_kv_attention_v1")
    return KvAttention(out, lse, mass)


def kv_evict(score, weights, table, lengths, keep: int, block_tokens: int = 16, sink: int = 1,
             recent: int = 1, decay: int = 0, stream=None) -> KvEviction:
    """Adds a step's block weights (float32 [seqs, kv_heads, width], as
    kv_attention returns them) to the accumulated score (int64 [seqs, width],
    2^30 to a unit of weight; `decay`: score >> decay is taken off first) and
    lets the blocks of least score beyond `keep` leave each table, never the
    first `sink` nor the last `recent`.  Returns the new score, table and
    lengths, the pages freed (in block order, -1 behind) and their counts;
    the inputs stay as they are."""
    index = table.get_device()
    _need(index >= 0, "the tensors have to be on a CUDA device")
    if not _here(index, stream):
        with _On(index, stream):
            return kv_evict(score, weights, table, lengths, keep, block_tokens, sink, recent, decay)
    import torch
    shape = seqs, width = _check_table(index, table, lengths, "lengths")
    _need(score.dtype == torch.int64 and score.shape == shape and score.is_contiguous()
          and score.get_device() == index, "score: int64 [seqs, width], contiguous")
    _need(weights.dtype == torch.float32 and weights.dim() == 3 and weights.shape[0] == seqs
          and weights.shape[2] == width and weights.is_contiguous()
          and weights.get_device() == index,
          "weights: float32 [seqs, kv_heads, width], contiguous")
    _need(not (keep | block_tokens | sink | recent | decay) >> 32,
          "keep, block_tokens, sink, recent and decay are counts of 32 bits")
    plain, like = torch.contiguous_format, torch.empty_like
    new_score = like(score)
    new_table, freed = like(table, memory_format=plain), like(table, memory_format=plain)
    new_lengths, freed_counts = like(lengths, memory_format=plain), like(lengths, memory_format=plain)
    batch = _EVICT.pack(_EVICT.size, 1, seqs, weights.shape[1], width, block_tokens, keep, sink,
                        recent, decay, score.data_ptr(), weights.data_ptr(), table.data_ptr(),
                        table.stride(0), lengths.data_ptr(), new_score.data_ptr(),
                        new_table.data_ptr(), new_lengths.data_ptr(), freed.data_ptr(),
                        freed_counts.data_ptr())
    check(_lib.load().hbfsim_kv_evict_v1(batch, _handle(index)), "hbfsim_kv_evict_v1")
    return KvEviction(new_score, new_table, new_lengths, freed, freed_counts)


def kv_verify(target, draft, tokens, accept, sample, counts=None, lengths=None,
              stream=None) -> KvVerified:
    """Drafted tokens against the target's probabilities, from given random numbers.

    target: [seqs, n + 1, vocab], float32, bfloat16 or float16; draft: what they were drawn from,
    [seqs, n, vocab] of the same type, or None for tokens that were looked up.  tokens: int32
    [seqs, n] (n at most 32).  accept: float32 [seqs, n], sample: float32 [seqs], uniform in [0, 1).
    counts: int32 [seqs], how many of its n drafts a sequence has (default: all).

    Token i is accepted while accept * draft < target at it.  The next token is drawn with `sample`
    from what target has over draft in the row of the first token that was not accepted (with no
    draft: from target without that token), or from the last row where all were.  Returns accepted
    (int32 [seqs]), tokens (int32 [seqs, n + 1]: those accepted, the next one, -1 behind) and,
    where `lengths` (int32 [seqs], with the drafted tokens) is given, the lengths without those that
    were not accepted; else None.  kv_resize gives back the pages behind them."""
    index = target.get_device()
    _need(index >= 0, "the tensors have to be on a CUDA device")
    if not _here(index, stream):
        with _On(index, stream):
            return kv_verify(target, draft, tokens, accept, sample, counts, lengths)
    import torch
    of = target.dtype
    kind = _lib.KV_P_F32 if of == torch.float32 else _lib.KV_P_BF16 if of == torch.bfloat16 else \
        _lib.KV_P_F16 if of == torch.float16 else None
    _need(kind is not None and target.dim() == 3 and target.shape[1] > 0 and target.shape[2] > 0,
          "target: float32, bfloat16 or float16 [seqs, n + 1, vocab]")
    seqs, rows, vocab = target.shape
    n = rows - 1
    by_seq, by_token, by_value = target.stride()
    _need(by_value == 1 or vocab == 1, "the last axis of target has to be contiguous")
    draft_at = draft_seq = draft_token = 0
    if draft is not None:
        _need(draft.dtype == target.dtype and draft.shape == (seqs, n, vocab)
              and draft.get_device() == index and (draft.stride(2) == 1 or vocab == 1 or n == 0),
              "draft: [seqs, n, vocab] of target's type on its device, the last axis contiguous")
        draft_seq, draft_token, _ = draft.stride()
        draft_at = draft.data_ptr() or 256  # 0: no draft
    per_draft, per_seq = (seqs, n), (seqs,)
    _need(tokens is not None and tokens.dtype == torch.int32 and tokens.shape == per_draft
          and tokens.get_device() == index and tokens.is_contiguous(),
          "tokens: int32 [seqs, n], contiguous, on target's device")
    _need(accept.dtype == torch.float32 and accept.shape == per_draft and accept.get_device() == index
          and accept.is_contiguous(), "accept: float32 [seqs, n], contiguous, on target's device")
    _need(sample.dtype == torch.float32 and sample.shape == per_seq and sample.get_device() == index
          and sample.is_contiguous(), "sample: float32 [seqs], contiguous, on target's device")
    _need(counts is None or counts.dtype == torch.int32 and counts.shape == per_seq
          and counts.get_device() == index and counts.is_contiguous(),
          "counts: int32 [seqs], contiguous, on target's device")
    _need(lengths is None or lengths.dtype == torch.int32 and lengths.shape == per_seq
          and lengths.get_device() == index and lengths.is_contiguous(),
          "lengths: int32 [seqs], contiguous, on target's device")
    _need(not (target.requires_grad or draft is not None and draft.requires_grad)
          or not torch.is_grad_enabled(), "no gradient passes through a draw: detach the tensors or "
          "call under torch.no_grad()")
    if lengths is None:
        accepted, kept, out = tokens.new_empty(seqs), None, tokens.new_empty((seqs, rows))
    else:
        accepted, kept, out = _parts(tokens, seqs, seqs, seqs * rows)
        out = out.view(seqs, rows)
    batch = _VERIFY.pack(_VERIFY.size, 1, kind, seqs, n, vocab, target.data_ptr(), by_seq, by_token,
                         draft_at, draft_seq, draft_token, tokens.data_ptr(), accept.data_ptr(),
                         sample.data_ptr(), counts.data_ptr() if counts is not None else 0,
                         lengths.data_ptr() if kept is not None else 0, accepted.data_ptr(),
                         out.data_ptr(), kept.data_ptr() if kept is not None else 0)
    check(_lib.load().hbfsim_kv_verify_v1(batch, _handle(index)), "hbfsim_kv_verify_v1")
    return KvVerified(accepted, out, kept)


def _parts(like, *sizes):
    """New tensors of `like`'s type and device, one after the other in one allocation."""
    return like.new_empty(sum(sizes)).unsafe_split_with_sizes(sizes)


def _check_pool(refs, table, index) -> None:
    import torch
    _need(refs.dtype == torch.int32 and refs.dim() == 1 and refs.is_contiguous()
          and refs.get_device() == index, "refs: int32 [pages] on the table's device, contiguous")


def kv_resize(refs, table, lengths, want, block_tokens: int = 16, freed=None, freed_counts=None,
              inplace: bool = False, stream=None) -> KvResized:
    """Every sequence gets or gives back pages, so that it can hold `want` tokens of which it holds
    `lengths` (int32 [seqs] both; want 0: the sequence is finished).

    refs: int32 [pages], how many table entries name a page; it is free below 1.  Entries behind
    `want` become -1 and their pages go back, and so do listed pages (freed, freed_counts: as
    kv_evict returns them).  Blocks that tokens from `lengths` on fall into get the lowest free
    pages, in order of sequence and block, where they have none or share theirs with others.

    Returns refs, table (new, or with `inplace` the arguments themselves, changed), limits (int32
    [seqs]: the tokens that a sequence may be filled up to; below `want` only if pages ran out) and
    src, dst (int32 [seqs]): the pages to copy with kv_copy before the append, for blocks that
    were shared and go on being filled; -1 for none."""
    index = table.get_device()
    _need(index >= 0, "the tensors have to be on a CUDA device")
    if not _here(index, stream):
        with _On(index, stream):
            return kv_resize(refs, table, lengths, want, block_tokens, freed, freed_counts, inplace)
    import torch
    seqs, width = _check_table(index, table, lengths, "lengths")
    _need(want.dtype == torch.int32 and want.shape == lengths.shape and want.is_contiguous()
          and want.get_device() == index, "want: int32 [seqs] on the table's device, contiguous")
    _check_pool(refs, table, index)
    _need(not block_tokens >> 32, "block_tokens is a count of 32 bits")
    freed_rows = freed_width = freed_at = freed_counts_at = 0
    if freed is not None:
        _need(freed_counts is not None and freed.dtype == torch.int32 and freed.dim() == 2
              and freed_counts.dtype == torch.int32 and freed_counts.shape == freed.shape[:1]
              and freed.is_contiguous() and freed_counts.is_contiguous()
              and freed.get_device() == index and freed_counts.get_device() == index,
              "freed: int32 [rows, width], freed_counts: int32 [rows], contiguous, on the table's device")
        freed_rows, freed_width = freed.shape
        freed_at, freed_counts_at = freed.data_ptr(), freed_counts.data_ptr()
    else:
        _need(freed_counts is None, "freed_counts without freed")
    if inplace:
        new_refs, new_table = refs, table
    else:
        new_refs = torch.empty_like(refs)
        new_table = torch.empty_like(table, memory_format=torch.contiguous_format)
    limits, src, dst = _parts(refs, seqs, seqs, seqs)
    batch = _RESIZE.pack(
        _RESIZE.size + _WORKSPACE.size, 1, seqs, width, block_tokens, freed_rows, freed_width, 0,
        refs.shape[0], refs.data_ptr(), table.data_ptr(), table.stride(0), lengths.data_ptr(),
        want.data_ptr(), freed_at, freed_counts_at, new_refs.data_ptr(), new_table.data_ptr(),
        new_table.stride(0), limits.data_ptr(), src.data_ptr(), dst.data_ptr())
    lib = _lib.load()
    size = lib.hbfsim_kv_resize_workspace_v1(batch + _NO_WORKSPACE)
    space = refs.new_empty(size // 4)
    check(lib.hbfsim_kv_resize_v1(batch + _WORKSPACE.pack(space.data_ptr(), size), _handle(index)),
          "hbfsim_kv_resize_v1")
    return KvResized(new_refs, new_table, limits, src, dst)


def kv_fork(refs, table, lengths, parents, block_tokens: int = 16, inplace: bool = False,
            stream=None) -> KvForked:
    """Sequences go on as children of others: row r of the new table is the row of parents[r]
    (int32 [rows]; outside [0, seqs): an empty row), as far as its length reaches.  Rows that no
    child goes on from give their pages back.  A block that is still filled is shared until
    kv_resize parts it.

    Returns refs (int32 [pages]; with `inplace` the argument itself, changed), the new table (int32
    [rows, width]) and lengths (int32 [rows])."""
    index = table.get_device()
    _need(index >= 0, "the tensors have to be on a CUDA device")
    if not _here(index, stream):
        with _On(index, stream):
            return kv_fork(refs, table, lengths, parents, block_tokens, inplace)
    import torch
    seqs, width = _check_table(index, table, lengths, "lengths")
    _check_pool(refs, table, index)
    _need(not block_tokens >> 32, "block_tokens is a count of 32 bits")
    _need(parents.dtype == torch.int32 and parents.dim() == 1 and parents.is_contiguous()
          and parents.get_device() == index, "parents: int32 [rows] on the table's device, contiguous")
    rows = parents.shape[0]
    new_refs = refs if inplace else torch.empty_like(refs)
    new_table, new_lengths = refs.new_empty((rows, width)), torch.empty_like(parents)
    batch = _FORK.pack(_FORK.size, 1, seqs, rows, width, block_tokens, refs.shape[0],
                       refs.data_ptr(), table.data_ptr(), table.stride(0), lengths.data_ptr(),
                       parents.data_ptr(), new_refs.data_ptr(), new_table.data_ptr(),
                       new_lengths.data_ptr())
    check(_lib.load().hbfsim_kv_fork_v1(batch, _handle(index)), "hbfsim_kv_fork_v1")
    return KvForked(new_refs, new_table, new_lengths)


def kv_copy(cache: KvCache, src, dst, source: KvCache | None = None, stream=None) -> None:
    """Page dst[i] of the cache becomes page src[i] of `source` (default: of the cache itself); src,
    dst: int32 [n], as kv_resize and kv_compact return them.  An entry outside its pool is passed
    over.  No page of dst may occur twice, nor among the pages that are read."""
    if not _here(cache.index, stream):
        with _On(cache.index, stream):
            return kv_copy(cache, src, dst, source)
    import torch
    source = cache if source is None else source
    _need(source.index == cache.index and source.kv_heads == cache.kv_heads
          and source.head_dim == cache.head_dim and source.block_tokens == cache.block_tokens,
          "source: pages of the same shape on the cache's device")
    for x in (src, dst):
        _need(x.dtype == torch.int32 and x.dim() == 1 and x.shape == src.shape
              and x.is_contiguous() and x.get_device() == cache.index,
              "src and dst: int32 [n], contiguous, on the cache's device")
    check(_lib.load().hbfsim_kv_copy_v1(source._packed, cache._packed, src.data_ptr(),
                                        dst.data_ptr(), src.shape[0], _handle(cache.index)),
          "hbfsim_kv_copy_v1")


def kv_compact(refs, table, inplace: bool = False, stream=None) -> KvCompacted:
    """The pages in use move to the front of the pool: the highest goes to the lowest free page, as
    long as there is a free one below.

    Returns refs and table after the moves (new, or with `inplace` the arguments themselves,
    changed), src and dst (int32 [pages // 2], -1 behind the moves: for kv_copy, on every layer's
    cache), live (int32 [1]: pages in use) and where (int32 [pages]: the new place of every page in
    use, -1 for the others; for other tables on the same pool)."""
    index = table.get_device()
    _need(index >= 0, "the tensors have to be on a CUDA device")
    if not _here(index, stream):
        with _On(index, stream):
            return kv_compact(refs, table, inplace)
    import torch
    shape = table.shape
    _need(len(shape) == 2 and table.dtype == torch.int32
          and (table.stride(1) == 1 or shape[1] <= 1 or shape[0] == 0),
          "table: int32 [seqs, width], rows contiguous")
    _check_pool(refs, table, index)
    seqs, width = shape
    pages = refs.shape[0]
    if inplace:
        new_refs, new_table = refs, table
    else:
        new_refs = torch.empty_like(refs)
        new_table = torch.empty_like(table, memory_format=torch.contiguous_format)
    lib = _lib.load()
    size = lib.hbfsim_kv_compact_workspace_v1(_COMPACT.pack(
        _COMPACT.size + _WORKSPACE.size, 1, seqs, width, pages, *[0] * 10) + _NO_WORKSPACE)
    # the workspace is small: some bytes for every warp
    space, src, dst, live = _parts(refs, size // 4, pages // 2, pages // 2, 1)
    where = torch.empty_like(refs)
    batch = _COMPACT.pack(
        _COMPACT.size + _WORKSPACE.size, 1, seqs, width, pages, refs.data_ptr(), table.data_ptr(),
        table.stride(0), new_refs.data_ptr(), new_table.data_ptr(), new_table.stride(0),
        src.data_ptr(), dst.data_ptr(), live.data_ptr(), where.data_ptr())
    check(lib.hbfsim_kv_compact_v1(batch + _WORKSPACE.pack(space.data_ptr(), size),
                                   _handle(index)), "hbfsim_kv_compact_v1")
    return KvCompacted(new_refs, new_table, src, dst, live, where)


def kv_block_reads(cache: KvCache, table, blocks, counts, base: int):
    """The cache reads of a list (as kv_select returns it) as an access batch:
    (address, bytes, op) device tensors for Context.submit, one access per
    listed block and head of its keys and values (2 * block_tokens * head_dim
    bytes, 4 KiB at 16 tokens of 128), in list order.  Page p, head h lies at
    base + (p * kv_heads + h) * block_bytes: the cache's own layout placed at
    `base` in the simulated address space.  An index that the table does not
    have, or whose page is not in the pool, is passed over, as the attention
    does."""
    import torch
    _need(blocks.dim() == 4 and table.dim() == 2 and table.shape[0] >= blocks.shape[0],
          "blocks: [seqs, tokens, kv_heads, top] with a row of the table for each of seqs")
    heads, top = blocks.shape[2:]
    width = table.shape[1]
    rank = torch.arange(top, device=blocks.device)
    listed = (rank < counts[..., None]) & (blocks >= 0) & (blocks < width)
    if width == 0:  # listed by no one
        page = torch.zeros_like(blocks, dtype=torch.int64)
    else:
        index = torch.where(listed, blocks, 0).long()
        page = torch.gather(table.long(), 1, index.flatten(1)).view_as(index)
    listed &= (page >= 0) & (page < cache.pages)
    head = torch.arange(heads, device=blocks.device)[:, None]
    address = base + (page * heads + head) * cache.block_bytes
    address = address[listed]
    return (address, torch.full_like(address, cache.block_bytes, dtype=torch.int32),
            torch.zeros_like(address, dtype=torch.uint8))
