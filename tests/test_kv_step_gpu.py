"""The operators around the attention together, as a server runs them: drafted tokens with rotary
positions on forked sequences, pages given, parted, taken back and compacted.  Everything but the
attention's floating outputs is equal to the oracle's at every step; the attention has the bounds of
test_kv_gpu.py."""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import attend_and_check, from_gpu, int32, same_cache, to_gpu, torch_

pytestmark = pytest.mark.gpu

HEADS, GROUP, DIM, BLOCK, DRAFTS, VOCAB = 2, 2, 64, 16, 3, 50


class Server:
    """The GPU's state and the oracle's, side by side."""

    def __init__(self, seqs, width, pages, seed):
        torch = torch_()
        from hbfsim_b200 import KvCache, KvRotary
        self.rng = np.random.default_rng(seed)
        self.gpu = KvCache.empty(pages, HEADS, DIM, BLOCK)
        self.cache = from_gpu(self.gpu)
        self.rotary = KvRotary.of(DIM, base=100.0, sections=(8, 12, 12))
        self.freq, self.axis = self.rotary.freq.cpu().numpy(), self.rotary.axis.cpu().numpy()
        self.refs, self.lengths = np.zeros(pages, np.int32), np.zeros(seqs, np.int32)
        self.table = np.full((seqs, width), -1, np.int32)
        self.torch = torch

    def same(self, got, want):
        for name, w in zip(got._fields, want):
            assert np.array_equal(getattr(got, name).cpu().numpy(), w), name

    def copy(self, src, dst):
        from hbfsim_b200 import kv_copy
        kv_copy(self.gpu, src, dst)
        for a, b in zip(src.cpu().numpy(), dst.cpu().numpy()):
            if a >= 0:
                for x in self.cache.values():
                    x[b] = x[a]

    def resize(self, want):
        from hbfsim_b200 import kv_resize
        got = kv_resize(int32(self.refs), int32(self.table), int32(self.lengths), int32(want), BLOCK)
        result = ko.resize(self.refs, self.table, self.lengths, want, BLOCK)
        self.same(got, result)
        self.refs, self.table, limits = result[:3]
        assert np.array_equal(limits, want)
        self.copy(got.src, got.dst)

    def append(self, count):
        """New tokens behind the lengths; returns the turned queries."""
        from hbfsim_b200 import kv_append_rotary
        torch, rng = self.torch, self.rng
        offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
        total = int(offsets[-1])
        new = lambda heads: torch.from_numpy(rng.standard_normal((total, heads, DIM))).to(torch.bfloat16).cuda()  # noqa: E731
        q, k, v = new(HEADS * GROUP), new(HEADS), new(HEADS)
        positions = rng.integers(0, 1000, (3, total)).astype(np.int32)
        out = kv_append_rotary(self.gpu, q, k, v, int32(self.table), int32(self.lengths), int32(positions),
                               self.rotary, offsets=int32(offsets))
        f32 = lambda t: t.float().cpu().numpy()  # noqa: E731
        want = torch.from_numpy(ko.rotate(f32(q), positions, self.freq, self.axis, False)).to(torch.bfloat16)
        assert torch.equal(out.cpu(), want)
        turned = ko.rotate(f32(k), positions, self.freq, self.axis, False).astype(np.float64)
        ko.append(self.cache, turned, v.double().cpu().numpy(), self.table, self.lengths, offsets)
        same_cache(self.gpu, self.cache)
        self.lengths = (self.lengths + count).astype(np.int32)
        return out

    def verify(self):
        from hbfsim_b200 import kv_verify
        torch, rng, seqs = self.torch, self.rng, len(self.lengths)
        soft = lambda x: x / x.sum(-1, keepdims=True)  # noqa: E731
        target = soft(np.exp(2 * rng.standard_normal((seqs, DRAFTS + 1, VOCAB)))).astype(np.float32)
        draft = soft(target[:, :DRAFTS] ** 0.8).astype(np.float32)
        tokens = np.array([[rng.choice(VOCAB, p=p / p.sum(dtype=np.float64)) for p in row.astype(np.float64)]
                           for row in draft], np.int32)
        accept, sample = rng.random((seqs, DRAFTS)).astype(np.float32), rng.random(seqs).astype(np.float32)
        cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
        got = kv_verify(cuda(target), cuda(draft), int32(tokens), cuda(accept), cuda(sample), lengths=int32(self.lengths))
        want = ko.verify(target, draft, tokens, accept, sample, [DRAFTS] * seqs, self.lengths)
        self.same(got, want)
        self.lengths = want[2]

    def fork(self, parents):
        from hbfsim_b200 import kv_fork
        got = kv_fork(int32(self.refs), int32(self.table), int32(self.lengths), int32(parents), BLOCK)
        result = ko.fork(self.refs, self.table, self.lengths, parents, BLOCK)
        self.same(got, result)
        self.refs, self.table, self.lengths = result

    def compact(self):
        from hbfsim_b200 import kv_compact
        got = kv_compact(int32(self.refs), int32(self.table))
        result = ko.compact(self.refs, self.table)
        self.same(got, result)
        self.refs, self.table = result[:2]
        self.copy(got.src, got.dst)


def test_drafted_steps_of_forked_sequences():
    server = Server(seqs=5, width=14, pages=90, seed=1)
    prompts = np.array([37, 5, 16, 90, 0], np.int32)
    server.resize(prompts)
    server.append(prompts)
    grew = np.zeros(5, np.int64)
    for step in range(16):
        if step % 4 == 1:
            server.fork(server.rng.integers(0, 5, 5).astype(np.int32))
        if step % 5 == 2:
            server.compact()
        seqs = len(server.lengths)
        server.resize((server.lengths + DRAFTS + 1).astype(np.int32))
        q = server.append(np.full(seqs, DRAFTS + 1))
        attend_and_check(server.cache, q.view(seqs, DRAFTS + 1, HEADS * GROUP, DIM), server.table, server.lengths,
                         gpu=server.gpu)
        before = server.lengths
        server.verify()
        assert (server.lengths <= before).all() and (server.lengths >= before - DRAFTS).all()
        grew += server.lengths > before - DRAFTS - 1
        counts = np.bincount(server.table[server.table >= 0], minlength=90)
        assert np.array_equal(server.refs, counts)
    assert (grew == 16).all()
    server.resize(np.zeros(5, np.int32))  # all finished
    assert not server.refs.any() and (server.table == -1).all()


def test_compaction_moves_what_attention_reads():
    torch = torch_()
    from hbfsim_b200 import kv_attention
    server = Server(seqs=4, width=8, pages=64, seed=2)
    server.resize(np.array([100, 60, 120, 128], np.int32))
    server.append(np.array([100, 60, 120, 128]))
    server.fork(np.array([3, 1], np.int32))
    q = torch.randn((2, 1, HEADS * GROUP, DIM), device="cuda").to(torch.bfloat16)
    read = lambda: kv_attention(server.gpu, q, int32(server.table), int32(server.lengths))  # noqa: E731
    before = read()
    server.compact()
    after = read()
    assert torch.equal(before.out, after.out) and torch.equal(before.lse, after.lse)
    assert (server.table[server.table >= 0] < (server.refs > 0).sum()).all()


def graph_inputs(rng, seqs, width, pages):
    torch = torch_()
    lengths = rng.integers(1, 40, seqs).astype(np.int32)
    table = np.full((seqs, width), -1, np.int32)
    order = rng.permutation(pages)
    at = 0
    for b in range(seqs):
        have = -(-int(lengths[b]) // BLOCK)
        table[b, :have] = order[at:at + have]
        at += have
    table[1] = table[0]
    lengths[1] = lengths[0]  # forked
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    qkv = torch.from_numpy(rng.standard_normal((seqs, 2, 8, DIM))).to(torch.bfloat16)
    target = rng.random((seqs, 2, VOCAB)).astype(np.float32)
    return dict(refs=torch.from_numpy(refs), table=torch.from_numpy(table), lengths=torch.from_numpy(lengths), qkv=qkv,
                places=torch.from_numpy(rng.integers(0, 900, (seqs, 2)).astype(np.int32)),
                target=torch.from_numpy(target / target.sum(-1, keepdims=True)),
                tokens=torch.from_numpy(rng.integers(0, VOCAB, (seqs, 1)).astype(np.int32)),
                accept=torch.from_numpy(rng.random((seqs, 1)).astype(np.float32)),
                sample=torch.from_numpy(rng.random(seqs).astype(np.float32)))


def step(s, cache, rotary):
    from hbfsim_b200 import kv_append_rotary, kv_compact, kv_copy, kv_fork, kv_resize, kv_verify
    room = kv_resize(s["refs"], s["table"], s["lengths"], s["lengths"] + 2, inplace=True)
    kv_copy(cache, room.src, room.dst)
    q = kv_append_rotary(cache, s["qkv"][:, :, :4], s["qkv"][:, :, 4:6], s["qkv"][:, :, 6:], s["table"], s["lengths"],
                         s["places"], rotary)
    kept = kv_verify(s["target"], None, s["tokens"], s["accept"], s["sample"], lengths=s["lengths"] + 2)
    child = kv_fork(s["refs"], s["table"], kept.lengths, kept.accepted)
    return [room.limits, room.src, room.dst, q, *kept, *child, *kv_compact(child.refs, child.table),
            s["refs"], s["table"], cache.data.view(torch_().uint8), cache.scale, cache.bounds]


def test_two_captured_graphs_of_one_step():
    """A step captured twice, on streams of their own, replayed in turn with new inputs: as run at
    once.  The graphs share nothing: outputs and workspaces are each one's own."""
    torch = torch_()
    from hbfsim_b200 import KvCache, KvRotary
    rng = np.random.default_rng(7)
    seqs, width, pages = 6, 5, 40
    rotary = KvRotary.of(DIM)
    captured = []
    for _ in range(2):
        s = {k: v.cuda() for k, v in graph_inputs(rng, seqs, width, pages).items()}
        cache = KvCache.empty(pages, HEADS, DIM, BLOCK)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s, cache, rotary)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(s, cache, rotary)
        captured.append((graph, s, cache, outs))
    for turn in range(4):
        wanted = []
        for graph, s, cache, outs in captured:
            new = graph_inputs(rng, seqs, width, pages)
            plain = {k: v.cuda() for k, v in new.items()}
            eager = KvCache.empty(pages, HEADS, DIM, BLOCK)
            wanted.append([x.clone() for x in step(plain, eager, rotary)])
            for k, v in new.items():
                s[k].copy_(v)
            cache.data.view(torch.uint8).zero_()
            cache.scale.fill_(1)
            cache.bounds.zero_()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(captured, streams):  # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, outs), want in zip(captured, wanted):
            for i, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), (turn, i)


def test_given_stream():
    """Work that a given stream has to wait for is waited for, and outputs belong to it."""
    torch = torch_()
    from hbfsim_b200 import (KvCache, KvRotary, kv_append_rotary, kv_compact, kv_copy, kv_fork, kv_resize, kv_verify)
    rng = np.random.default_rng(8)
    new = graph_inputs(rng, 6, 5, 40)
    plain = {k: v.cuda() for k, v in new.items()}
    rotary = KvRotary.of(DIM)
    eager = KvCache.empty(40, HEADS, DIM, BLOCK)
    want = [x.clone() for x in step(plain, eager, rotary)]
    side = torch.cuda.Stream()
    late = {k: torch.zeros_like(v, device="cuda") for k, v in new.items()}
    cache = KvCache.empty(40, HEADS, DIM, BLOCK)
    host = {k: v.pin_memory() for k, v in new.items()}
    busy = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(30):
            busy += 1  # keeps the stream occupied
        for k, v in host.items():
            late[k].copy_(v, non_blocking=True)
        more = late["lengths"] + 2
    room = kv_resize(late["refs"], late["table"], late["lengths"], more, inplace=True, stream=side)
    kv_copy(cache, room.src, room.dst, stream=side)
    q = kv_append_rotary(cache, late["qkv"][:, :, :4], late["qkv"][:, :, 4:6], late["qkv"][:, :, 6:], late["table"],
                         late["lengths"], late["places"], rotary, stream=side)
    kept = kv_verify(late["target"], None, late["tokens"], late["accept"], late["sample"], lengths=more, stream=side)
    child = kv_fork(late["refs"], late["table"], kept.lengths, kept.accepted, stream=side)
    small = kv_compact(child.refs, child.table, stream=side)
    torch.cuda.synchronize()
    got = [room.limits, room.src, room.dst, q, *kept, *child, *small, late["refs"], late["table"],
           cache.data.view(torch.uint8), cache.scale, cache.bounds]
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i
