from .manager import RELEASED, CacheManager, CannotShare, OutOfPages, OutOfSlots, PagedGroup, PagePool, StateGroup
from .storage import CacheStorage, PagedLayerView, StateLayerView
