from .errors import CacheCapacityError, CacheError, CacheOwnershipError
from .manager import CacheManager, CacheOrder, CacheStats, RequestCache
from .pools import IndexPool

__all__ = ["CacheCapacityError", "CacheError", "CacheOwnershipError", "CacheManager", "CacheOrder",
           "CacheStats", "RequestCache", "IndexPool"]
