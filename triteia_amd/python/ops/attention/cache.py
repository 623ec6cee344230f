"""The paged cache of keys and values: made, written without rotation, and read back."""
import torch

from triteia_amd.python import capi
from triteia_amd.python.capi import PagedCache

__all__ = ["PagedCache", "paged_cache", "cache_write", "cache_read"]


def paged_cache(n_pages, kv_heads, dim, page=64, dtype=torch.float16, device="cuda"):
    """An empty PagedCache in fp16, bf16, int8 or float8_e4m3fn (the 8-bit types with one float32 scale for every token and head)."""
    k, v = (torch.zeros((n_pages, kv_heads, page, dim), dtype=dtype, device=device) for _ in range(2))
    scales = [torch.zeros((n_pages, kv_heads, page), dtype=torch.float32, device=device) for _ in range(2)] if k.element_size() == 1 else []
    return PagedCache(k, v, *scales)


def cache_write(cache, k, v, slots):
    """k, v [tokens, kv_heads, dim] into the cache at `slots` (int32 / int64 [tokens], distinct; outside the cache: not written).  In 8 bits a row's scale
    puts its largest magnitude at the end of the codes' range; a row that holds an infinity or a NaN reads back as NaN."""
    capi.rotary_cache(None, k, v, None, None, cache, slots)


def cache_read(cache, slots, dtype=None):
    """(k, v) [len(slots), kv_heads, dim] as the values that the cache holds at `slots`, in `dtype` (the cache's own, or fp16 from 8 bits, if None); zeros
    where a slot lies outside the cache."""
    return capi.cache_read(cache, slots, dtype or (cache.dtype if cache.kind == 0 else torch.float16))
