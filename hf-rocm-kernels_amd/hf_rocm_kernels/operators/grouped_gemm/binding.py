from typing import Optional

import torch
from torch import Tensor

import hf_rocm_kernels._HFRK_C  # noqa: F401  (registers torch.ops._HFRK_C)


def _grouped_gemm(a: Tensor, b: Tensor, scale_a: Tensor, scale_b: Optional[Tensor], offsets: Tensor, rows: Optional[Tensor], output: Tensor) -> None:
    torch.ops._HFRK_C.grouped_gemm(a, b, scale_a, scale_b, offsets, rows, output)
