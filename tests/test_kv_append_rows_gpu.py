"""kv_append of few and of many tokens whose rows begin on 16 bytes and off them, at every number of
channels: equal to its definition."""
import numpy as np
import pytest

import kv_oracle as ko
from test_kv_gpu import int32, make_table, random_cache, same_cache, to_gpu, torch_, type_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("dim,block,heads,kind", [(64, 16, 3, "bf16"), (128, 32, 2, "f16"), (256, 16, 2, "bf16"),
                                                  (256, 64, 1, "f16")])
def test_rows_on_and_off_16_bytes(dim, block, heads, kind, odd):
    torch = torch_()
    from hbfsim_b200 import kv_append
    rng = np.random.default_rng(dim + block + odd)
    what = [(s, n) for s in (0, 1, 9, block - 1) for n in (1, 2, 3, 4, 5, 8, 16, 20, 2 * block + 3)]
    start, count = (np.array(x, np.int32) for x in zip(*what))
    offsets = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    pages = int((-(-(start + count) // block)).sum()) + 1
    cache = random_cache(rng, pages, heads, block, dim)
    table = make_table(rng, start + count, block, pages)
    x = rng.standard_normal((int(offsets[-1]), 2 * heads, dim + odd)) * 10.0 ** rng.uniform(-3, 3, (int(offsets[-1]), 1, 1))
    kv = torch.from_numpy(x).to(type_of(kind)).cuda()[..., odd:]
    k, v = kv[:, :heads], kv[:, heads:]
    gpu = to_gpu(cache)
    kv_append(gpu, k, v, int32(table), int32(start), offsets=int32(offsets))
    ko.append(cache, k.double().cpu().numpy(), v.double().cpu().numpy(), table, start, offsets)
    same_cache(gpu, cache)
