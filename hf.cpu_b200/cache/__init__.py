from .pages import CacheGroup, KVCacheManager, LayerCache, OutOfPages, PagePool, eight_bits_refusal
from .slots import OutOfSlots, StateSlots

__all__ = ["PagePool", "CacheGroup", "KVCacheManager", "LayerCache", "OutOfPages", "StateSlots", "OutOfSlots", "eight_bits_refusal"]
