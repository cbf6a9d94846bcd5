from typing import Optional

import torch
from torch import Tensor

import hf_rocm_kernels._HFRK_C  # noqa: F401  (registers torch.ops._HFRK_C)


def _tree_attention(
    query: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, lengths: Tensor, starts: Optional[Tensor], mask: Optional[Tensor],
    scale: float, key_scale: Optional[Tensor], value_scale: Optional[Tensor], out_scale: Optional[Tensor], output: Tensor,
) -> None:
    torch.ops._HFRK_C.tree_attention(query, key_cache, value_cache, page_table, lengths, starts, mask, scale, key_scale, value_scale, out_scale,
                                     output)
