"""Operators over a paged key/value cache held in 8 bits (include/hbfsim/kv_v1.h).

One decode step of a layer is

    kv_append(cache, k, v, table, start)                 # the new tokens' keys and values
    pick = kv_select(cache, q, table, lengths, top=128)  # blocks worth reading, per head
    got = kv_attention(cache, q, table, lengths, blocks=pick.blocks,
                       counts=pick.counts, weights=True)
    rest = kv_evict(score, got.weights, table, lengths, keep=...)
    reads = kv_block_reads(cache, table, pick.blocks, pick.counts, base)  # for Context.submit

kv_attention without lists reads every block.  Arguments that do not fit
raise ValueError here, or HbfsimError from the C ABI.  Calls are asynchronous
on `stream` (default: torch's current stream); outputs and workspace belong
to that stream.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

from . import _lib
from ._lib import check
from .api import _stream_handle

__all__ = ["KvCache", "KvAttention", "KvSelection", "KvEviction", "kv_append", "kv_attention",
           "kv_select", "kv_evict", "kv_block_reads"]


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
                 "device", "_struct", "_ref")

    def __init__(self, data, scale, bounds):
        import torch
        _need(data.dim() == 5 and data.shape[2] == 2 and data.dtype == torch.float8_e4m3fn,
              "data: float8_e4m3fn [pages, kv_heads, 2, block_tokens, head_dim]")
        self.pages, self.kv_heads, _, self.block_tokens, self.head_dim = data.shape
        head = (self.pages, self.kv_heads, 2)
        _need(scale.dtype == torch.float32 and tuple(scale.shape) == head,
              "scale: float32 [pages, kv_heads, 2]")
        _need(bounds.dtype == torch.int8 and tuple(bounds.shape) == head + (self.head_dim,),
              "bounds: int8 [pages, kv_heads, 2, head_dim]")
        _need(data.is_contiguous() and scale.is_contiguous() and bounds.is_contiguous(),
              "data, scale and bounds have to be contiguous")
        self.device = data.device
        _need(data.is_cuda and scale.device == data.device and bounds.device == data.device,
              "data, scale and bounds have to be on one CUDA device")
        self.data, self.scale, self.bounds = data, scale, bounds
        self._struct = _lib.KvCacheV1(ctypes.sizeof(_lib.KvCacheV1), 1, self.kv_heads,
                                      self.head_dim, self.block_tokens, 0, self.pages,
                                      data.data_ptr(), scale.data_ptr(), bounds.data_ptr())
        self._ref = ctypes.addressof(self._struct)

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


def _check_table(cache_device, table, per_seq, names):
    import torch
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.device == cache_device
          and (table.shape[1] <= 1 or table.stride(1) == 1),
          "table: int32 [seqs, width] on the cache's device, rows contiguous")
    for x, name in zip(per_seq, names):
        _need(x.dim() == 1 and x.dtype == torch.int32 and x.shape[0] == table.shape[0]
              and x.device == cache_device and (x.shape[0] <= 1 or x.stride(0) == 1),
              f"{name}: int32 [seqs] on the cache's device, contiguous")


class _On:
    """Makes the device and the stream current for the allocations of a call."""

    __slots__ = ("device", "stream", "guard", "context")

    def __init__(self, device, stream):
        self.device, self.stream = device, stream

    def __enter__(self):
        import torch
        self.guard = self.context = None
        if self.device.index is not None and self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        if self.stream is not None:
            _need(self.stream.device == self.device, "the stream is of another device")
            self.context = torch.cuda.stream(self.stream)
            self.context.__enter__()
        return _stream_handle(self.stream)

    def __exit__(self, *exc):
        if self.context is not None:
            self.context.__exit__(*exc)
        if self.guard is not None:
            self.guard.__exit__(*exc)


def kv_append(cache: KvCache, k, v, table, start, offsets=None, stream=None) -> None:
    """Quantises new tokens into the blocks of their sequences.

    k, v: [seqs, n, kv_heads, head_dim], or with `offsets` (int32 [seqs + 1])
    ragged [tokens, kv_heads, head_dim], sequence s owning tokens
    [offsets[s], offsets[s + 1]); any strides with a contiguous last axis.
    start: int32 [seqs], tokens a sequence held before.  Writes data, scale
    and bounds of the touched blocks in place."""
    import torch
    _check_table(cache.device, table, (start,), ("start",))
    seqs, width = table.shape
    _need(k.shape == v.shape and k.dtype == v.dtype and k.device == v.device == cache.device
          and k.dim() == (4 if offsets is None else 3)
          and k.shape[-2:] == (cache.kv_heads, cache.head_dim),
          "k and v: one shape and type, [seqs, n, kv_heads, head_dim] or with offsets "
          "[tokens, kv_heads, head_dim], on the cache's device")
    if offsets is None:
        _need(k.shape[0] == seqs, "k: as many sequences as the table")
        k, v = k.flatten(0, 1), v.flatten(0, 1)  # a copy where one stride cannot serve both axes
    else:
        _need(offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.shape[0] == seqs + 1
              and offsets.device == cache.device and offsets.is_contiguous(),
              "offsets: int32 [seqs + 1] on the cache's device, contiguous")
    tokens = k.shape[0]
    if tokens == 0:
        return
    _need(k.stride(-1) == 1 and v.stride(-1) == 1, "the last axis of k and v has to be contiguous")
    batch = _lib.KvAppendBatchV1(ctypes.sizeof(_lib.KvAppendBatchV1), 1, _type(k), seqs, width, 0,
                                 tokens, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                                 v.stride(0), v.stride(1), table.data_ptr(), table.stride(0),
                                 start.data_ptr(), 0 if offsets is None else offsets.data_ptr())
    with _On(cache.device, stream) as handle:
        check(_lib.load().hbfsim_kv_append_v1(cache._ref, ctypes.addressof(batch), handle),
              "hbfsim_kv_append_v1")


def _query(cache: KvCache, q, table, lengths):
    _check_table(cache.device, table, (lengths,), ("lengths",))
    _need(q.dim() == 4 and q.shape[0] == table.shape[0] and q.shape[3] == cache.head_dim
          and q.device == cache.device, "q: [seqs, tokens, q_heads, head_dim] on the cache's device")
    _need(q.shape[2] > 0 and q.shape[2] % cache.kv_heads == 0,
          "q_heads has to be a multiple of kv_heads")
    _need(q.stride(3) == 1, "the last axis of q has to be contiguous")
    return _lib.KvQueryV1(ctypes.sizeof(_lib.KvQueryV1), 1, _type(q), q.shape[0], q.shape[1],
                          q.shape[2], table.shape[1], 0, q.data_ptr(), q.stride(0), q.stride(1),
                          q.stride(2), table.data_ptr(), table.stride(0), lengths.data_ptr())


def kv_select(cache: KvCache, q, table, lengths, top: int, sink: int = 1, recent: int = 1,
              stream=None) -> KvSelection:
    """For every query token and key/value head the blocks worth reading: the
    first `sink`, the last `recent` and those whose bounds allow the largest
    products with the group's queries, `top` in all.

    q: [seqs, tokens, q_heads, head_dim], the newest tokens, which `lengths`
    counts.  Returns blocks (int32 [seqs, tokens, kv_heads, top], ascending,
    -1 behind the count) and counts (int32 [seqs, tokens, kv_heads])."""
    import torch
    query = _query(cache, q, table, lengths)
    lib = _lib.load()
    with _On(cache.device, stream) as handle:
        shape = (q.shape[0], q.shape[1], cache.kv_heads)
        blocks = torch.empty(shape + (max(0, top),), dtype=torch.int32, device=cache.device)
        counts = torch.empty(shape, dtype=torch.int32, device=cache.device)
        ref = ctypes.addressof(query)
        size = lib.hbfsim_kv_select_workspace_v1(cache._ref, ref)
        space = torch.empty(size, dtype=torch.uint8, device=cache.device)
        check(lib.hbfsim_kv_select_v1(cache._ref, ref, max(0, top), max(0, sink), max(0, recent),
                                      blocks.data_ptr(), counts.data_ptr(), space.data_ptr(),
                                      size, handle), "hbfsim_kv_select_v1")
    return KvSelection(blocks, counts)


def kv_attention(cache: KvCache, q, table, lengths, scale: float | None = None, blocks=None,
                 counts=None, weights: bool = False, stream=None) -> KvAttention:
    """Attention of the newest tokens: q [seqs, tokens, q_heads, head_dim],
    token t at position lengths - tokens + t.  scale: of the products
    (default head_dim ** -0.5).  blocks, counts: lists as kv_select returns
    them (default: every block).

    Returns out (q's type and shape), lse (float32 [seqs, tokens, q_heads],
    natural logarithm of the sum of exponentials) and, if asked for, weights
    (float32 [seqs, kv_heads, width]: softmax weight of every block, summed
    over the group's heads and the tokens; else None)."""
    import torch
    query = _query(cache, q, table, lengths)
    top = 0
    if blocks is not None:
        shape = (q.shape[0], q.shape[1], cache.kv_heads)
        _need(counts is not None and blocks.dtype == torch.int32 and counts.dtype == torch.int32
              and blocks.dim() == 4 and tuple(blocks.shape[:3]) == shape
              and tuple(counts.shape) == shape and blocks.is_contiguous()
              and counts.is_contiguous() and blocks.device == counts.device == cache.device,
              "blocks and counts: int32 [seqs, tokens, kv_heads(, top)] on the cache's device, "
              "contiguous")
        top = blocks.shape[3]
        _need(top > 0, "a list has to have room for one block")
    else:
        _need(counts is None, "counts without blocks")
    lib = _lib.load()
    with _On(cache.device, stream) as handle:
        out = torch.empty(q.shape, dtype=q.dtype, device=cache.device)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=cache.device)
        mass = None
        if weights:
            mass = torch.empty((q.shape[0], cache.kv_heads, table.shape[1]), dtype=torch.float32,
                               device=cache.device)
            if q.shape[1] == 0:
                mass.zero_()
        args = _lib.KvAttentionArgsV1(
            ctypes.sizeof(_lib.KvAttentionArgsV1), 1,
            1.0 / math.sqrt(cache.head_dim) if scale is None else scale, top,
            None if blocks is None else blocks.data_ptr() or 16,
            None if blocks is None else counts.data_ptr() or 16, out.data_ptr(), lse.data_ptr(),
            mass.data_ptr() if weights else None, None, 0)
        ref, query_ref = ctypes.addressof(args), ctypes.addressof(query)
        args.workspace_bytes = lib.hbfsim_kv_attention_workspace_v1(cache._ref, query_ref, ref)
        space = torch.empty(args.workspace_bytes, dtype=torch.uint8, device=cache.device)
        args.workspace = space.data_ptr()
        check(lib.hbfsim_kv_attention_v1(cache._ref, query_ref, ref, handle),
              "hbfsim_kv_attention_v1")
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
    import torch
    _check_table(table.device, table, (lengths,), ("lengths",))
    seqs, width = table.shape
    _need(table.is_cuda, "the tensors have to be on a CUDA device")
    _need(score.dtype == torch.int64 and tuple(score.shape) == (seqs, width)
          and score.is_contiguous() and score.device == table.device,
          "score: int64 [seqs, width], contiguous")
    _need(weights.dtype == torch.float32 and weights.dim() == 3 and weights.shape[0] == seqs
          and weights.shape[2] == width and weights.is_contiguous()
          and weights.device == table.device,
          "weights: float32 [seqs, kv_heads, width], contiguous")
    lib = _lib.load()
    with _On(table.device, stream) as handle:
        got = KvEviction(torch.empty_like(score),
                         torch.empty((seqs, width), dtype=torch.int32, device=table.device),
                         torch.empty(seqs, dtype=torch.int32, device=table.device),
                         torch.empty((seqs, width), dtype=torch.int32, device=table.device),
                         torch.empty(seqs, dtype=torch.int32, device=table.device))
        batch = _lib.KvEvictBatchV1(
            ctypes.sizeof(_lib.KvEvictBatchV1), 1, seqs, weights.shape[1], width, block_tokens,
            max(0, keep), max(0, sink), max(0, recent), max(0, decay), score.data_ptr(),
            weights.data_ptr(), table.data_ptr(), table.stride(0), lengths.data_ptr(),
            got.score.data_ptr(), got.table.data_ptr(), got.lengths.data_ptr(),
            got.freed.data_ptr(), got.freed_counts.data_ptr())
        check(lib.hbfsim_kv_evict_v1(ctypes.addressof(batch), handle), "hbfsim_kv_evict_v1")
    return got


def kv_block_reads(cache: KvCache, table, blocks, counts, base: int):
    """The cache reads of a list (as kv_select returns it) as an access batch:
    (address, bytes, op) device tensors for Context.submit, one access per
    listed block and head of its keys and values (2 * block_tokens * head_dim
    bytes, 4 KiB at 16 tokens of 128), in list order.  Page p, head h lies at
    base + (p * kv_heads + h) * block_bytes: the cache's own layout placed at
    `base` in the simulated address space."""
    import torch
    seqs, tokens, heads, top = blocks.shape
    rank = torch.arange(top, device=blocks.device)
    listed = rank < counts[..., None]
    index = torch.where(listed, blocks, 0).long()
    page = torch.gather(table.long(), 1, index.view(seqs, -1)).view_as(index)
    listed &= (page >= 0) & (page < cache.pages)
    head = torch.arange(heads, device=blocks.device)[:, None]
    address = base + (page * heads + head) * cache.block_bytes
    address = address[listed]
    return (address, torch.full_like(address, cache.block_bytes, dtype=torch.int32),
            torch.zeros_like(address, dtype=torch.uint8))
