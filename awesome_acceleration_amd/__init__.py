"""MI355X-native (gfx950) attention hot path for the Qwen3 serving engine.

Drop-in replacements for the reference engine's ``flash_attn`` calls and its
``index_copy_`` KV store, implemented by hand-written HIP kernels in
``libaac_attn.so`` (C ABI: include/aac_attn.h).
"""
from .flash_attn_interface import (  # noqa: F401
    decode_paged,
    flash_attn_func,
    flash_attn_varlen_func,
    flash_attn_with_kvcache,
    kv_store,
    varlen_prefill_with_kvcache,
)
from .kv4 import (  # noqa: F401
    alloc_kv4_cache,
    decode_paged_kv4,
    flash_attn_with_kv4cache,
    kv4_export,
    kv4_import,
    kv4_load,
    kv4_store,
    qk_norm_rope_store_kv4,
)
from .paged import BlockAllocator, SlotCacheManager  # noqa: F401

__version__ = "0.1.0"
