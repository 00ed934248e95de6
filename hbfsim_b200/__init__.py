"""B200-native batched HBF access-timing path (HBFSim hot path).

The CUDA library libhbfsim_b200.so (hbfsim_b200/csrc) holds the kernels and
the C ABI; this package is the Python host side.  Importing it does not load
the library; `Context` does, and fails loudly if it is missing.
"""
from .api import (BatchResult, Context, HbfsimError, link_batch, link_profiles,  # noqa: F401
                  prefetch_sweep, submit_linked)
from .kv import (KvAttention, KvCache, KvCompacted, KvEviction, KvForked,  # noqa: F401
                 KvResized, KvRotary, KvSelection, KvVerified, kv_append, kv_append_rotary,
                 kv_attention, kv_block_reads, kv_compact, kv_copy, kv_evict, kv_fork, kv_resize,
                 kv_select, kv_verify)
from ._lib import (ACCESS_BYPASS, ACCESS_FOREIGN, ACCESS_MODELED,  # noqa: F401
                   ACCESS_UNSUPPORTED, MODEL_DIE, MODEL_FAST, MODEL_HYBRID,
                   MODEL_REFERENCE, RANGE_CAPACITY, RANGE_TIMING)
