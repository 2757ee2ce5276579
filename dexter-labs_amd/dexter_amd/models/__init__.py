"""Callers of the attention path: the per-layer KV caches and a self-attention layer."""

from .kv_cache import KVCache
from .paged_kv_cache import PagedKVCache
from .attention import SelfAttention

__all__ = ["KVCache", "PagedKVCache", "SelfAttention"]
