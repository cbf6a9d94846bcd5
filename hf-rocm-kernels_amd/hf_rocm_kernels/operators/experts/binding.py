from typing import Optional

import torch
from torch import Tensor

import hf_rocm_kernels._HFRK_C  # noqa: F401  (registers torch.ops._HFRK_C)


def _route_experts(
    logits: Tensor, top_k: int, bias: Optional[Tensor], sigmoid: bool, renormalize: bool, factor: float, mask: Optional[Tensor],
    weights: Tensor, experts: Tensor, places: Tensor, rows: Tensor, offsets: Tensor,
) -> None:
    torch.ops._HFRK_C.route_experts(logits, top_k, bias, sigmoid, renormalize, factor, mask, weights, experts, places, rows, offsets)


def _combine_experts(y: Tensor, weights: Tensor, places: Tensor, base: Optional[Tensor], output: Tensor) -> None:
    torch.ops._HFRK_C.combine_experts(y, weights, places, base, output)
