"""kv_verify through the C ABI with `accepted` in counts' memory and `lengths_out` in that of lengths:
what it gives with outputs of their own."""
import ctypes

import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import int32, torch_

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,vocab", [(300, 40), (3, 40000)])  # one thread block to a sequence, and eight
def test_counts_and_lengths_in_place(seqs, vocab):
    torch = torch_()
    from hbfsim_b200 import _lib
    rng = np.random.default_rng(seqs)
    n = 3
    target = rng.random((seqs, n + 1, vocab)).astype(np.float32)
    target /= target.sum(-1, keepdims=True)
    tokens = rng.integers(0, vocab, (seqs, n)).astype(np.int32)
    accept = (rng.random((seqs, n)) / vocab).astype(np.float32)
    sample = rng.random(seqs).astype(np.float32)
    counts, lengths = rng.integers(-1, n + 2, seqs).astype(np.int32), rng.integers(10, 99, seqs).astype(np.int32)
    want = ko.verify(target, None, tokens, accept, sample, counts, lengths)
    cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    t, x, u, s, c, l = cuda(target), cuda(tokens), cuda(accept), cuda(sample), int32(counts), int32(lengths)
    out = torch.empty((seqs, n + 1), dtype=torch.int32, device="cuda")
    batch = _lib.KvVerifyBatchV1(
        struct_size=ctypes.sizeof(_lib.KvVerifyBatchV1), version=1, type=_lib.KV_P_F32, seqs=seqs, drafts=n, vocab=vocab,
        target=t.data_ptr(), target_stride_seq=t.stride(0), target_stride_token=t.stride(1), tokens=x.data_ptr(),
        accept=u.data_ptr(), sample=s.data_ptr(), counts=c.data_ptr(), lengths=l.data_ptr(), accepted=c.data_ptr(),
        tokens_out=out.data_ptr(), lengths_out=l.data_ptr())
    rc = _lib.load().hbfsim_kv_verify_v1(ctypes.byref(batch), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert rc == 0
    for got, w in zip((c, out, l), want):
        assert np.array_equal(got.cpu().numpy(), w)
