from torch import Tensor
import torch

import hf_rocm_kernels._HFRK_C  # noqa: F401  (registers torch.ops._HFRK_C)


def _rotary(x: Tensor, positions: Tensor, frequencies: Tensor, magnitude: float, interleaved: bool, output: Tensor) -> None:
    torch.ops._HFRK_C.rotary(x, positions, frequencies, magnitude, interleaved, output)
