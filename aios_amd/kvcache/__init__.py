from .base import BaseKVCache
from .mha_pool import MHAKVCache
from .mha_pool8 import MHAKVCache8

__all__ = ["BaseKVCache", "MHAKVCache", "MHAKVCache8"]
