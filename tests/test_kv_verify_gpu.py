"""kv_verify against its definition in whole numbers and fractions (oracle/kv_oracle.py): equal."""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import int32, torch_

pytestmark = pytest.mark.gpu


def types():
    torch = torch_()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def check(target, draft, tokens, accept, sample, counts=None, lengths=None, stream=None):
    """target, draft: CUDA tensors; the others numpy.  Compares with the oracle."""
    torch = torch_()
    from hbfsim_b200 import kv_verify
    seqs, rows, _ = target.shape
    f32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()  # noqa: E731
    got = kv_verify(target, draft, int32(tokens).view(seqs, rows - 1), f32(accept).view(seqs, rows - 1), f32(sample),
                    counts=None if counts is None else int32(counts),
                    lengths=None if lengths is None else int32(lengths), stream=stream)
    torch.cuda.synchronize()
    host = lambda x: x.double().cpu().numpy()  # noqa: E731
    want = ko.verify(host(target), None if draft is None else host(draft), np.asarray(tokens).reshape(seqs, rows - 1),
                     np.asarray(accept, np.float32).reshape(seqs, rows - 1), np.asarray(sample, np.float32),
                     [rows - 1] * seqs if counts is None else counts, [0] * seqs if lengths is None else lengths)
    assert got.accepted.cpu().tolist() == want[0].tolist(), "accepted"
    assert got.tokens.cpu().tolist() == want[1].tolist(), "tokens"
    if lengths is None:
        assert got.lengths is None
    else:
        assert got.lengths.cpu().tolist() == want[2].tolist(), "lengths"
    return got


def make(rng, seqs, n, vocab, kind, drafted, sharp=2.0):
    """Target and draft probabilities that mostly agree; tokens from the draft."""
    torch = torch_()
    soft = lambda x: np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)  # noqa: E731
    logits = sharp * rng.standard_normal((seqs, n + 1, vocab))
    draft = soft(logits[:, :n] + 0.5 * rng.standard_normal((seqs, n, vocab)))
    target = torch.from_numpy(soft(logits)).to(types()[kind]).cuda()
    tokens = np.array([[rng.choice(vocab, p=draft[b, i]) for i in range(n)] for b in range(seqs)], np.int32).reshape(seqs, n)
    draft = torch.from_numpy(draft).to(types()[kind]).cuda() if drafted else None
    accept = rng.random((seqs, n)).astype(np.float32)
    if not drafted:
        accept *= 0.3 / max(1, vocab) ** 0.5
    return target, draft, tokens, accept, rng.random(seqs).astype(np.float32)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("seqs,n,vocab", [(1, 3, 8), (40, 4, 50), (5, 1, 1), (9, 2, 3), (7, 32, 33), (3, 15, 1000),
                                          (2, 0, 257), (64, 3, 700)])
def test_verify(seqs, n, vocab, kind, drafted):
    rng = np.random.default_rng(seqs * 1000 + n * 100 + vocab)
    args = make(rng, seqs, n, vocab, kind, drafted)
    lengths = rng.integers(0, 5000, seqs)
    check(*args)
    counts = rng.integers(-2, n + 3, seqs)  # some below 0 or past n
    check(*args, counts=counts, lengths=lengths)


@pytest.mark.parametrize("vocab,seqs", [(4096, 3), (8191, 2), (32768, 1), (65537, 2), (100003, 1), (131072, 2)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_verify_large_vocabularies(vocab, seqs, kind):
    """Rows that one to eight thread blocks share; the border at the beginning, the end and between
    two blocks' slices."""
    rng = np.random.default_rng(vocab)
    target, draft, tokens, accept, sample = make(rng, seqs, 2, vocab, kind, True)
    check(target, draft, tokens, accept, sample)
    for s in (0.0, 1 - 2.0 ** -24, 0.125, 0.5, 0.875):
        check(target, draft, tokens, accept * 0 + 0.999, np.full(seqs, s))
        check(target, None, tokens, accept * 0 + 0.999, np.full(seqs, s))


def test_many_sequences():
    """More sequences than thread blocks are resident."""
    rng = np.random.default_rng(2)
    check(*make(rng, 1500, 2, 40, "f32", True), counts=np.arange(1500) % 3, lengths=np.arange(1500))


def test_views_and_odd_strides():
    """Rows inside a wider tensor, at odd elements; sequences in reverse is a copy's business."""
    torch = torch_()
    rng = np.random.default_rng(3)
    target, draft, tokens, accept, sample = make(rng, 4, 3, 777, "f32", True)
    wide = torch.zeros((4, 4, 1000), device="cuda")
    wide[:, :, 5:782] = target
    deep = torch.zeros((3, 4, 777), device="cuda")
    deep.copy_(draft.transpose(0, 1))
    check(wide[:, :, 5:782], deep.transpose(0, 1), tokens, accept, sample)
    assert not check(target, draft, tokens, accept, sample).tokens.requires_grad
    # aligned rows whose last elements are no whole load
    even = torch.zeros((4, 4, 1024), device="cuda")
    even[:, :, :777] = target
    check(even[:, :, :777], even[:, :3, :777], tokens, accept, sample)


def test_special_values():
    """Probabilities that are zero, one, subnormal, negative, above one, infinite or NaN; random
    numbers at and past the ends; tokens outside the vocabulary; rows of zeros."""
    torch = torch_()
    vocab = 6
    nan, inf = float("nan"), float("inf")
    rows = torch.tensor([
        [0, 0, 0, 0, 0, 0], [0, 0, 1, 0, 0, 0], [nan, 0.5, inf, -1, 0.25, 1e-40], [-inf, 2, 0, 0, 0, 0],
        [2.0 ** -41, 2.0 ** -40, 3 * 2.0 ** -41, 0, 0, 0], [0.25, 0.25, 0.25, 0.25, 0, 0], [1, 1, 1, 1, 1, 1]])
    pairs = [(a, b) for a in range(len(rows)) for b in range(len(rows))]
    for token in (0, 2, 5, -1, vocab, -2 ** 31):
        for u in (0.0, 0.3, 1 - 2.0 ** -24, 1.0, nan, -1.0, inf):
            target = torch.stack([torch.stack([rows[a], rows[b]]) for a, b in pairs]).cuda()
            draft = torch.stack([rows[b][None] for a, b in pairs]).cuda()
            n = len(pairs)
            for q in (draft, None):
                check(target, q, np.full((n, 1), token), np.full((n, 1), u), np.full(n, u))


def test_equal_target_and_draft_accepts_all_but_never_ties():
    """u * q < p: with p == q every u below 1 accepts; with u q == p exactly it does not."""
    torch = torch_()
    p = torch.full((1, 3, 4), 0.25, device="cuda")
    got = check(p, p[:, :2].contiguous(), [[1, 3]], [[1 - 2.0 ** -24, 0.0]], [0.6])
    assert got.accepted.item() == 2 and got.tokens.tolist() == [[1, 3, 2]]
    q = torch.full((1, 2, 4), 0.5, device="cuda")
    assert check(p, q, [[1, 3]], [[0.5, 0.0]], [0.6]).accepted.item() == 0


def test_no_sequences():
    torch = torch_()
    got = check(torch.zeros((0, 3, 8), device="cuda"), None, np.zeros((0, 2)), np.zeros((0, 2)), np.zeros(0))
    assert got.tokens.shape == (0, 3)


@pytest.mark.parametrize("bad", ["type", "draft type", "draft shape", "tokens", "long", "accept", "sample", "counts",
                                 "many", "gradient", "strides", "cpu", "no tokens"])
def test_refusals(bad):
    torch = torch_()
    from hbfsim_b200 import HbfsimError, kv_verify
    n = 33 if bad == "many" else 2
    p = torch.full((1, n + 1, 8), 0.125, device="cuda")
    call = dict(target=p, draft=p[:, :n], tokens=int32(np.zeros((1, n))), accept=torch.zeros((1, n), device="cuda"),
                sample=torch.zeros(1, device="cuda"))
    if bad == "type":
        call["target"] = p.double()
    elif bad == "draft type":
        call["draft"] = call["draft"].half()
    elif bad == "draft shape":
        call["draft"] = p
    elif bad == "tokens":
        call["tokens"] = int32(np.zeros((1, 3)))
    elif bad == "long":
        call["tokens"] = call["tokens"].long()
    elif bad == "accept":
        call["accept"] = call["accept"].double()
    elif bad == "sample":
        call["sample"] = torch.zeros(2, device="cuda")
    elif bad == "counts":
        call["counts"] = int32([1, 2])
    elif bad == "gradient":
        call["target"] = p.clone().requires_grad_()
    elif bad == "strides":
        call["target"] = p.transpose(1, 2).contiguous().transpose(1, 2)
    elif bad == "cpu":
        call["tokens"] = call["tokens"].cpu()
    elif bad == "no tokens":
        call["tokens"] = None
    with pytest.raises((ValueError, HbfsimError)):
        kv_verify(**call)


def test_rows_past_32_bit_offsets():
    """The largest vocabulary, rows that begin behind 2^31 elements."""
    torch = torch_()
    from hbfsim_b200 import kv_verify
    vocab, seqs = 1 << 22, 180
    target = torch.zeros((seqs, 3, vocab), device="cuda")
    target[:, :, 7] = 0.25
    target[-1, 0, vocab - 1] = 0.5
    target[-1, 1, 100] = 0.75
    tokens = np.full((seqs, 2), 7, np.int32)
    tokens[-1] = [vocab - 1, 3]
    one = torch.full((seqs, 2), 0.3, device="cuda")
    got = kv_verify(target, None, int32(tokens), one, torch.full((seqs,), 0.9, device="cuda"))
    assert got.accepted.tolist() == [0] * (seqs - 1) + [1]
    # all weight lies on the token that was not accepted: the target alone counts
    assert got.tokens[:-1].tolist() == [[7, -1, -1]] * (seqs - 1)
    assert got.tokens[-1].tolist() == [vocab - 1, 100, -1]
