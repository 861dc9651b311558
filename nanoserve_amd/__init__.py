"""nanoserve_amd: MI355X-native paged attention for nanoserve.

The package replaces the GPU side of nanoserve's attention op and KV-cache
write with hand-written gfx950 HIP kernels behind a C ABI
(include/nanoserve_paged.h), keeping the reference's call contract:

  attn_fn(query, k_cache, v_cache, md, scale) -> out   (paged_attention_hip)
  PagedKVCache.write(layer, key, value, slot_mapping)  (reshape_and_cache)
  BlockSpaceManager.slot_mapping(seq, start, end)      (addressing contract)
  rotary.apply + PagedKVCache.write fused              (rope_reshape_and_cache)

Beside the reference's: the same write and attention over a cache held in 4
bits (kv4.py), and the draw of a token from given uniform numbers
(sampling.sample_rows).
"""

from .attention import AttentionMetadata, get_attention_backend, paged_attention_hip
from .block_manager import BlockSpaceManager
from .kv_cache import PagedKVCache, kv_bytes_per_token, reshape_and_cache
from .kv4 import (Int4PagedKVCache, gather_cache_int4, paged_attention_int4, reshape_and_cache_int4,
                  rope_reshape_and_cache_int4)
from .rotary import RotaryEmbedding, rope_reshape_and_cache
from .sampling import argmax_rows, sample_rows

__version__ = "0.1.0"

__all__ = [
    "AttentionMetadata",
    "BlockSpaceManager",
    "Int4PagedKVCache",
    "PagedKVCache",
    "argmax_rows",
    "gather_cache_int4",
    "get_attention_backend",
    "kv_bytes_per_token",
    "paged_attention_hip",
    "paged_attention_int4",
    "reshape_and_cache",
    "reshape_and_cache_int4",
    "RotaryEmbedding",
    "rope_reshape_and_cache",
    "rope_reshape_and_cache_int4",
    "sample_rows",
]
