from typing import Optional

import torch
from torch import Tensor

import hf_rocm_kernels._HFRK_C  # noqa: F401  (registers torch.ops._HFRK_C)


def _int8_gemm(a: Tensor, b: Tensor, output: Tensor, base: Optional[Tensor], scale_a: Tensor, scale_b: Optional[Tensor]) -> None:
    torch.ops._HFRK_C.int8_gemm(a, b, output, base, scale_a, scale_b)
