from .fp4 import FP4KVCache
from .pool import MHAKVCache

__all__ = ["FP4KVCache", "MHAKVCache"]
