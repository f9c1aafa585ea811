"""bpt — B200-native paged-KV GQA decode attention (sm_100a CUDA behind a C ABI).

Public API (the reference project's ``bpt`` names are kept where they exist):

  paged_decode_attention(q, k_cache, v_cache, block_table, seq_lens, scale=None,
                         num_splits=None)              FP16 cache
  bpt.triton_fp16.paged_decode_attention_triton        the reference's name for the same call
  bpt.evict   paged_decode_attention_scored, append_tokens, select_evictions, compact_cache,
              evict_tokens                             bounded fp16 / bf16 caches
  bpt.diff    paged_decode_attention_diff              differential decode attention
  bpt.cache.build_paged_cache                          reference test-cache builder (torch)
  bpt.roofline                                         bytes-per-token / roofline model + CLI

There is no CPU or Triton fallback: compute entry points need CUDA tensors and the in-tree
library ``bpt/libbpt_b200.so`` (built by ``kvq-decode_b200/build.py``).
"""
from ._lib import BptArgumentError, BptError, BptUnsupportedError
from .cache import build_paged_cache
from .decode import choose_num_splits, paged_decode_attention
from .diff import paged_decode_attention_diff
from .evict import append_tokens, evict_tokens, paged_decode_attention_scored

__all__ = ["paged_decode_attention", "paged_decode_attention_scored",
           "paged_decode_attention_diff", "append_tokens", "evict_tokens", "choose_num_splits",
           "build_paged_cache", "BptError", "BptArgumentError", "BptUnsupportedError"]
__version__ = "0.1.0"
