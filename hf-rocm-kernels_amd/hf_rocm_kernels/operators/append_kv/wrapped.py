from typing import Optional

import torch
from torch import Tensor

from ...utils.dispatch import runs_now
from ..rotary.wrapped import heads_checks, rotation_checks
from .binding import _append_kv

_append_kv_new = torch.ops._HFRK_C.append_kv_new.default


def cache_checks(key_cache: Tensor, value_cache: Tensor, kv_heads: int, head_dim: int, dtype: torch.dtype, device: torch.device) -> None:
    for name, cache in (("key_cache", key_cache), ("value_cache", value_cache)):
        assert cache.dim() == 4 and tuple(cache.shape[2:]) == (kv_heads, head_dim), \
            f"Expected {name} to have shape (pages, page_size, {kv_heads}, {head_dim}) but got {cache.shape}"
        assert cache.dtype in (dtype, torch.float8_e4m3fn), f"Expected {name} to be {dtype} or torch.float8_e4m3fn but got {cache.dtype}"
        assert head_dim <= 1 or cache.stride(3) == 1, f"Expected {name} to have unit stride along head_dim but got {cache.stride()}"
        assert cache.size(1) >= 1, f"Expected {name} to have pages of one place or more but got {cache.shape}"
        assert cache.device == device, f"Expected {name} to be on {device} but got {cache.device}"
    assert key_cache.shape == value_cache.shape and key_cache.dtype == value_cache.dtype, "Expected key_cache and value_cache to have one shape and dtype"


def scale_checks(key_scale: Optional[Tensor], value_scale: Optional[Tensor], kv_heads: int, cache: Tensor) -> None:
    for name, scale in (("key_scale", key_scale), ("value_scale", value_scale)):
        if scale is not None:
            assert cache.dtype == torch.float8_e4m3fn, f"Expected no {name} for a cache of {cache.dtype}"
            assert scale.numel() in (1, kv_heads) and scale.dtype == torch.float32 and scale.is_contiguous(), \
                f"Expected {name} to be 1 or {kv_heads} contiguous float32 values but got {scale.shape} {scale.dtype}"
            assert scale.device == cache.device, f"Expected {name} to be on {cache.device} but got {scale.device}"


def append_kv_checks(
    key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor, slots: Tensor, positions: Optional[Tensor], frequencies: Optional[Tensor],
    query: Optional[Tensor], query_output: Optional[Tensor], key_scale: Optional[Tensor], value_scale: Optional[Tensor],
) -> None:
    heads_checks("key", key)
    heads_checks("value", value)
    tokens, kv_heads, head_dim = key.shape
    assert value.shape == key.shape and value.dtype == key.dtype, f"Expected value like key but got {value.shape = } {value.dtype = }"
    assert kv_heads >= 1, f"Expected one key head or more but got {key.shape = }"
    cache_checks(key_cache, value_cache, kv_heads, head_dim, key.dtype, key.device)
    assert slots.shape == (tokens,) and slots.dtype in (torch.int32, torch.int64) and slots.is_contiguous(), \
        f"Expected slots to be {tokens} contiguous int32 or int64 values but got {slots.shape} {slots.dtype}"
    assert (positions is None) == (frequencies is None), "Expected positions and frequencies together"
    if frequencies is not None:
        rotation_checks(tokens, head_dim, positions, frequencies, key.device)
    assert query is not None or query_output is None, "Expected query_output with a query only"
    if query is not None:
        assert frequencies is not None, "Expected frequencies and positions with a query"
        heads_checks("query", query)
        assert query.size(0) == tokens and query.size(2) == head_dim and query.dtype == key.dtype, \
            f"Expected query to have key's tokens, head_dim and dtype but got {query.shape = } {query.dtype = }"
        assert query_output.shape == query.shape and query_output.dtype == query.dtype, \
            f"Expected query_output like query but got {query_output.shape = } {query_output.dtype = }"
        assert query.device == key.device and query_output.device == key.device, f"Expected query and query_output to be on {key.device}"
    scale_checks(key_scale, value_scale, kv_heads, key_cache)
    assert value.device == key.device and slots.device == key.device, f"Expected value and slots to be on {key.device}"
    assert key.device.type == "cuda", f"Expected key.device to be of type cuda, but got {key.device.type = } instead."


def append_kv(
    key: Tensor,
    value: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    slots: Tensor,
    positions: Optional[Tensor] = None,
    frequencies: Optional[Tensor] = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
    query: Optional[Tensor] = None,
    query_output: Optional[Tensor] = None,
    key_scale: Optional[Tensor] = None,
    value_scale: Optional[Tensor] = None,
) -> Optional[Tensor]:
    """Appends a step's keys and values to a paged cache in one launch, the keys rotated on the way; a step's queries are rotated along with them.
    Args:
        - key, value: 16-bit (bfloat16 or float16) tensors of shape (tokens, kv_heads, head_dim), unit stride along head_dim: slices of a
            projection's output as they are
        - key_cache, value_cache: (pages, page_size, kv_heads, head_dim) of the same dtype or float8_e4m3fn, unit stride along head_dim and any
            other strides (a heads-major cache is passed transposed); modified in place
        - slots: (tokens, ) int32 or int64, page * page_size + place of each token; negative ones and those behind the last page are padding, and
            not written.  Two tokens in one slot leave values of either there
        - positions, frequencies, interleaved, magnitude: as in `rotary`; None: keys are stored as they are
        - query: (tokens, heads, head_dim), rotated into query_output (None: a new tensor; query itself: in place)
        - key_scale, value_scale: for float8_e4m3fn caches, positive float32 tensors of one value or one per key head: x / scale is stored,
            saturating at +-448, NaN kept; None: 1
    The caches and query_output may share memory with nothing else that the call takes (slices of one tensor that lie between each other do not); refused
    otherwise.  Inference only: the rotated queries carry no gradient.
    Outputs:
        - the rotated queries, None without a query
    """
    if query_output is None and runs_now(key):
        done, output = _append_kv_new(key, value, key_cache, value_cache, slots, positions, frequencies, magnitude, interleaved, query, key_scale,
                                      value_scale)  # one native operator; not done: what is wrong, say the checks
        if done:
            return output
    if query is not None and query_output is None:
        query_output = torch.empty(size=query.shape, dtype=query.dtype, device=query.device)
    append_kv_checks(key, value, key_cache, value_cache, slots, positions, frequencies, query, query_output, key_scale, value_scale)
    _append_kv(key, value, key_cache, value_cache, slots, positions, frequencies, magnitude, interleaved, query, query_output, key_scale,
               value_scale)
    return query_output
