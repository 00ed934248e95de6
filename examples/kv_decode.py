"""What a decode step reads from High-Bandwidth Flash, with real attention.

One layer of a paged 8-bit KV cache lies in a simulated HBF range: page p,
head h at base + (p * kv_heads + h) * block_bytes, 4 KiB each at 16 tokens of
128 channels.  Every step appends a token per sequence, lists the blocks worth
reading per head (kv_select), attends over them (kv_attention), lets the
blocks of least accumulated attention weight go (kv_evict), and times two
traces on the per-die model: the reads of the lists, and the reads that
attention over every block would have made.

    python examples/kv_decode.py --seqs 16 --context 4096 --steps 32 --top 64 --keep 200
"""
from __future__ import annotations

import argparse
import json
import sys
import tempfile
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from hbfsim_b200 import (Context, KvCache, RANGE_TIMING, kv_append, kv_attention,  # noqa: E402
                         kv_block_reads, kv_evict, kv_select)
from hbfsim_b200 import workloads as wl  # noqa: E402


def read_time(ctx: Context, cache: KvCache, table, blocks, counts) -> tuple[int, int]:
    """(ns, reads) of one step's block reads, all arriving when the last step's are done."""
    address, nbytes, op = kv_block_reads(cache, table, blocks, counts, wl.RANGE_BASE)
    start = ctx.simulated_time()
    timed = ctx.submit(address, nbytes, op, torch.full_like(address, start))
    return int(timed.done_ns.max()) - start, address.numel()


def run(seqs: int, context: int, steps: int, top: int, keep: int, q_heads: int = 32,
        kv_heads: int = 8, head_dim: int = 128, block: int = 16, seed: int = 0) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16)

    width = -(-(context + steps) // block)
    keep = min(keep, width)
    cache = KvCache.empty(seqs * width, kv_heads, head_dim, block)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(seqs * width, generator=gen, device="cuda").to(torch.int32).tolist()

    with tempfile.TemporaryDirectory() as tmp:
        work = wl.c1_workload()  # the profile of the decode workloads: 4 stacks of 16 channels
        size = -(-cache.data.numel() // wl.GIB) * wl.GIB
        listed = Context(work.write_profile(tmp), report_dir=tmp + "/listed")
        every = Context(work.write_profile(tmp), report_dir=tmp + "/every")
        for ctx in (listed, every):
            ctx.set_geometry(stacks=work.stacks, stripe_bytes=work.stripe_bytes)
            ctx.register_device(wl.RANGE_BASE, size, mode=RANGE_TIMING, permissions=3)

        # the prompts
        blocks = -(-context // block)
        for b in range(seqs):
            table[b, :blocks] = torch.tensor([free.pop() for _ in range(blocks)])
        zero = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        channel = torch.exp(0.5 * torch.randn((kv_heads, head_dim), generator=gen, device="cuda"))
        for at in range(0, context, 4096):  # in chunks: start grows
            n = min(4096, context - at)
            k = (normal(seqs, n, kv_heads, head_dim) * channel).to(torch.bfloat16)
            kv_append(cache, k, normal(seqs, n, kv_heads, head_dim), table, zero + at)

        lengths = zero + context
        score = torch.zeros((seqs, width), dtype=torch.int64, device="cuda")
        total = {"steps": steps, "listed_ns": 0, "every_ns": 0, "listed_reads": 0, "every_reads": 0,
                 "evicted_blocks": 0}
        for _ in range(steps):
            full = (lengths % block == 0).nonzero().flatten().tolist()
            for b in full:  # a new block begins
                table[b, int(lengths[b]) // block] = free.pop()
            q = normal(seqs, 1, q_heads, head_dim)
            k = (normal(seqs, 1, kv_heads, head_dim) * channel).to(torch.bfloat16)
            kv_append(cache, k, normal(seqs, 1, kv_heads, head_dim), table, lengths)
            lengths = lengths + 1

            pick = kv_select(cache, q, table, lengths, top=top)
            got = kv_attention(cache, q, table, lengths, blocks=pick.blocks, counts=pick.counts,
                               weights=True)
            ns, reads = read_time(listed, cache, table, pick.blocks, pick.counts)
            total["listed_ns"] += ns
            total["listed_reads"] += reads

            have = (-(-lengths // block))[:, None, None].expand(seqs, 1, kv_heads)
            all_blocks = torch.arange(width, dtype=torch.int32, device="cuda")
            ns, reads = read_time(every, cache, table,
                                  all_blocks.expand(seqs, 1, kv_heads, width), have)
            total["every_ns"] += ns
            total["every_reads"] += reads

            rest = kv_evict(score, got.weights, table, lengths, keep=keep, block_tokens=block,
                            decay=8)
            score, table, lengths = rest.score, rest.table, rest.lengths
            for b, n in enumerate(rest.freed_counts.tolist()):
                free += rest.freed[b, :n].tolist()
                total["evicted_blocks"] += n
        for ctx in (listed, every):
            ctx.close()
    assert torch.isfinite(got.out).all()
    total["listed_us_per_step"] = round(total.pop("listed_ns") / steps / 1e3, 3)
    total["every_us_per_step"] = round(total.pop("every_ns") / steps / 1e3, 3)
    return total


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("seqs", 16), ("context", 4096), ("steps", 32), ("top", 64), ("keep", 200)):
        p.add_argument(f"--{name}", type=int, default=value)
    result = run(**vars(p.parse_args(argv)))
    print(json.dumps(result))
    return result


if __name__ == "__main__":
    main()
