from .kv import CacheGroup, KVNeed, KVView, SequenceCache, StateNeed
from .prefix import PrefixGroups
from .slots import CacheFull, FreeList

__all__ = ["CacheFull", "CacheGroup", "FreeList", "KVNeed", "KVView", "PrefixGroups", "SequenceCache", "StateNeed"]
