from typing import Optional

import torch
from torch import Tensor

import hf_rocm_kernels._HFRK_C  # noqa: F401  (registers torch.ops._HFRK_C)


def _append_kv(
    key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor, slots: Tensor, positions: Optional[Tensor], frequencies: Optional[Tensor],
    magnitude: float, interleaved: bool, query: Optional[Tensor], query_output: Optional[Tensor], key_scale: Optional[Tensor],
    value_scale: Optional[Tensor],
) -> None:
    torch.ops._HFRK_C.append_kv(key, value, key_cache, value_cache, slots, positions, frequencies, magnitude, interleaved, query, query_output,
                                key_scale, value_scale)
