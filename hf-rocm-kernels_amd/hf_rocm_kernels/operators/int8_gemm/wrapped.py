from typing import Optional

import torch
from torch import Tensor

from ...utils.dispatch import runs_now
from .binding import _int8_gemm

_int8_linear = torch.ops._HFRK_C.int8_linear.default
_OUT_DTYPES = (torch.bfloat16, torch.float16)
MAX_K = 131056  # sums of 2^14 k stay within 32 bits


def int8_gemm_checks(a: Tensor, b: Tensor, scale_a: Tensor, scale_b: Optional[Tensor], base: Optional[Tensor], output: Tensor) -> None:
    # Check shapes
    assert a.dim() == 2, f"Expected a to have 2 dimensions but got {a.dim() = } instead."
    assert b.dim() == 2 and a.size(1) == b.size(0), f"Expected {a.shape = } and {b.shape = } to be (m, k) and (k, n)."
    (m, k), n = a.shape, b.size(1)
    assert k % 16 == 0 and 0 < k <= MAX_K, f"Expected {k = } to be a multiple of 16 from 16 to {MAX_K}"
    assert 1 <= n <= 1 << 21, f"Expected {n = } to be between 1 and 2^21"
    assert output.shape == (m, n), f"{output.shape} does not match with {a.shape = } and {b.shape = }"
    assert scale_a.numel() in (1, m), f"Expected scale_a to have 1 or {m} elements but got {scale_a.shape}"
    assert scale_b is None or scale_b.numel() in (1, n), f"Expected scale_b to have 1 or {n} elements but got {scale_b.shape}"
    # Check dtypes
    assert a.dtype == torch.int8 and b.dtype == torch.int8, f"Expected {a.dtype = } and {b.dtype = } to be torch.int8"
    assert output.dtype in _OUT_DTYPES, f"Expected {output.dtype = } to be torch.bfloat16 or torch.float16"
    for name, scale in (("scale_a", scale_a), ("scale_b", scale_b)):
        assert scale is None or scale.dtype == torch.float32, f"Expected {name} to be torch.float32 but got {scale.dtype}"
        assert scale is None or scale.is_contiguous(), f"Expected {name} to be contiguous"
    # Check layouts
    assert a.is_contiguous(), f"Expected a to be contiguous but got {a.stride() = }"
    assert b.stride(0) == 1, f"Expected b to be column-major but got {b.stride() = }"
    assert n == 1 or (b.stride(1) >= k and b.stride(1) % 16 == 0 and b.stride(1) <= 1 << 21), \
        f"Expected b's columns to be a multiple of 16 bytes apart, at least {k}: {b.stride() = }"
    assert output.is_contiguous(), f"Expected output to be contiguous but got {output.stride() = }"
    if base is not None:
        assert base.shape in ((n,), (m, n)), f"Expected base to be ({n},) or ({m}, {n}) but got {base.shape}"
        assert base.dtype == output.dtype and base.is_contiguous(), f"Expected base to be contiguous and {output.dtype} but got {base.dtype}"
    # Check devices
    device = a.device
    assert device.type == "cuda", f"Expected a.device to be of type cuda, but got {device.type = } instead."
    for name, t in (("b", b), ("scale_a", scale_a), ("scale_b", scale_b), ("base", base), ("output", output)):
        assert t is None or t.device == device, f"Expected {name} to be on {device} but got {t.device}"


def int8_gemm(
    a: Tensor,
    b: Tensor,
    scale_a: Tensor,
    scale_b: Optional[Tensor] = None,
    base: Optional[Tensor] = None,
    output: Optional[Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> Tensor:
    """base + scale_a * scale_b * (a @ b) on int8 codes, from one row to whole prompts (2^24): the sums are exact, scales and addend are applied in fp32, and the result
    is rounded once.
    Args:
        - a: an (m, k) int8 tensor in row-major format, k a multiple of 16 up to 131056
        - b: a (k, n) int8 tensor in column-major format (the `.t()` of an (n, k) weight), columns a multiple of 16 bytes apart
        - scale_a: float32, one or one per row of a (`quantize_int8` and `swiglu_dynamic` give these); scale_b: one, one per column of b, or None: 1
        - base: an addend of the result's dtype, (m, n) (a residual) or (n,) (a bias)
        - output: a tensor to write to (it may be base), or None for a new one of out_dtype (bfloat16 or float16)
    Where few tiles have a long k a call takes a workspace from torch's allocator (64 MiB at most).  Inference only: the result carries no gradient.
    """
    if output is None and a.dim() == 2 and b.dim() == 2 and runs_now(a) and a.dtype == torch.int8:
        row = base is not None and base.shape == b.shape[1:]
        if base is None or row or base.shape == (a.size(0), b.size(1)):  # (a linear's residual may have any shape of m * n elements, and its bias be none)
            out = _int8_linear(a, b.t(), scale_b, scale_a, base if row else None, None if row else base, out_dtype)
            if out is not None:  # one native operator; None: what is wrong, say the checks
                return out
    if output is None:
        output = torch.empty(size=(a.size(0), b.size(1)), dtype=out_dtype, device=a.device)
    int8_gemm_checks(a, b, scale_a, scale_b, base, output)
    _int8_gemm(a, b, output, base, scale_a, scale_b)
    return output
