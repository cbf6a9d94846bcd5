"""Torch form of the product, for callers who want to check the kernel.  The operator never calls it."""
from typing import Optional

import torch
from torch import Tensor


def reference_int8_gemm(a: Tensor, b: Tensor, scale_a: Tensor, scale_b: Optional[Tensor] = None, base: Optional[Tensor] = None) -> Tensor:
    """base + scale_a * scale_b * (a @ b) in 64 bits (the sums of codes are exact there)."""
    out = (a.double() @ b.double()) * scale_a.double().reshape(-1, 1)
    if scale_b is not None:
        out = out * scale_b.double().reshape(1, -1)
    return out if base is None else out + base.double()
