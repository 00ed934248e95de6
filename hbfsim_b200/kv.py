"""Operators over a paged key/value cache held in 8 bits (include/hbfsim/kv_v1.h).

One decode step of a layer is

    kv_append(cache, k, v, table, start)                 # the new tokens' keys and values
    pick = kv_select(cache, q, table, lengths, top=128)  # blocks worth reading, per head
    got = kv_attention(cache, q, table, lengths, blocks=pick.blocks,
                       counts=pick.counts, weights=True)
    rest = kv_evict(score, got.weights, table, lengths, keep=...)
    reads = kv_block_reads(cache, table, pick.blocks, pick.counts, base)  # for Context.submit

kv_attention without lists reads every block.  Arguments that do not fit
raise ValueError here, or HbfsimError from the C ABI; so do keys, values and
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

__all__ = ["KvCache", "KvAttention", "KvSelection", "KvEviction", "kv_append", "kv_attention",
           "kv_select", "kv_evict", "kv_block_reads"]

# The C structures of kv_v1.h as packed bytes (no padding: 8-byte fields lie at multiples of 8);
# _lib has the same structures field by field.
_CACHE = struct.Struct("<6I4Q")
_APPEND = struct.Struct("<6I3Q4qQq2Q")
_QUERY = struct.Struct("<8IQ3qQqQ")
_ATTENTION = struct.Struct("<2IfI7Q")
_EVICT = struct.Struct("<10I3Qq6Q")


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
          and (table.stride(1) == 1 or shape[1] <= 1),
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
        return
    k_token, k_head, k_dim = k.stride()
    v_token, v_head, v_dim = v.stride()
    _need(k_dim == 1 and v_dim == 1, "the last axis of k and v has to be contiguous")
    batch = _APPEND.pack(_APPEND.size, 1, _type(k), seqs, width, 0, tokens, k.data_ptr(),
                         v.data_ptr(), k_token, k_head, v_token, v_head, table.data_ptr(),
                         table.stride(0), start.data_ptr(), at)
    check(_lib.load().hbfsim_kv_append_v1(cache._packed, batch, _handle(cache.index)),
          "hbfsim_kv_append_v1")


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
