from .attnres import attnres_mix, attnres_mix_step
from .store import store_cache, store_cache8

__all__ = ["attnres_mix", "attnres_mix_step", "store_cache", "store_cache8"]
