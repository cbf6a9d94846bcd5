from typing import Optional, Tuple

import torch
from torch import Tensor

from ...utils.fp8 import amax_scale, fp8_quantize
from ...utils.int8 import int8_quantize, int8_scale


def reference_quantize_fp8(x: Tensor, scale_tensor: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """Torch form of `quantize_fp8`: the reference's fp8_quantize recipe (hf_rocm_kernels/utils/fp8.py:6-29, OCP
    flavour) with the given scale, or with one scale per row, amax/448."""
    if scale_tensor is None:
        scale_tensor = amax_scale(x, dim=1)
    q, _ = fp8_quantize(x, scale_tensor)
    return q, scale_tensor.reshape(-1)


def reference_quantize_int8(x: Tensor, scale_tensor: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """Torch form of `quantize_int8`: codes and the given scale, or one per row, amax/127 (NaN for a row that holds an infinity or a NaN)."""
    if scale_tensor is None:
        scale_tensor = int8_scale(x, dim=1)
        scale_tensor = torch.where(torch.isfinite(x.float()).all(dim=1, keepdim=True), scale_tensor, torch.nan)
    return int8_quantize(x, scale_tensor), scale_tensor.reshape(-1)
