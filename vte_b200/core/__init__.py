from .paged_cache import PagedKVCache
from .split_kv_attention import SplitKVAttentionDispatcher

__all__ = ["PagedKVCache", "SplitKVAttentionDispatcher"]
