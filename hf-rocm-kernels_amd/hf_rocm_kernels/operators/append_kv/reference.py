"""Torch form of the append, for callers who want to check the kernel.  The operators never call it."""
from typing import Optional

import torch
from torch import Tensor

from ..rotary.reference import reference_rotary


def reference_append_kv(
    key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor, slots: Tensor, positions: Optional[Tensor] = None,
    frequencies: Optional[Tensor] = None, interleaved: bool = False, magnitude: float = 1.0, query: Optional[Tensor] = None,
    key_scale: Optional[Tensor] = None, value_scale: Optional[Tensor] = None,
) -> Optional[Tensor]:
    """`append_kv` as a chain of torch calls, into the given caches; returns the rotated queries.  (Synchronises: slots outside the cache are taken out.)"""
    pages, page_size = key_cache.shape[:2]
    kept = (slots >= 0) & (slots < pages * page_size)
    where = slots[kept] // page_size, slots[kept] % page_size
    wide = torch.promote_types(key.dtype, torch.float32)
    key, value = key.to(wide), value.to(wide)
    if frequencies is not None:
        key = reference_rotary(key, positions, frequencies, interleaved, magnitude)
        query = None if query is None else reference_rotary(query, positions, frequencies, interleaved, magnitude)
    for cache, rows, scale in ((key_cache, key, key_scale), (value_cache, value, value_scale)):
        rows = rows[kept]
        if cache.dtype == torch.float8_e4m3fn:
            rows = rows if scale is None else rows * (1.0 / scale).reshape(1, -1, 1)
            cache.view(torch.uint8)[where] = rows.clamp(-448, 448).to(cache.dtype).view(torch.uint8)
        else:
            cache[where] = rows.to(cache.dtype)
    return query
