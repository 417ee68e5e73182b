"""Slots, paged keys and values, fixed-size per-sequence state."""
from .sequence_cache import (CacheError, FreeList, KV_FORMATS, KVEntry, KVGroup, QuantizedKVEntry,  # noqa: F401
                             SequenceCache, StateEntry, StateGroup, round_up)
