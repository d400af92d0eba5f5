from .block_pool import BlockPool, NoFreePages, chain_hash
from .manager import CacheManager, Fork, RequestCache, NoFreeSlot
from .device import DeviceCache, CacheView

__all__ = ["BlockPool", "NoFreePages", "chain_hash", "CacheManager", "Fork", "RequestCache", "NoFreeSlot",
           "DeviceCache", "CacheView"]
