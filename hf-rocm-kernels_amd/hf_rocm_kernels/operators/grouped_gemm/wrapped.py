from typing import Optional

import torch
from torch import Tensor

from ... import _capi
from ...utils.dispatch import runs_now
from ..int8_gemm.wrapped import MAX_K
from .binding import _grouped_gemm

_grouped_gemm_new = torch.ops._HFRK_C.grouped_gemm_new.default
_OUT_DTYPES = (torch.bfloat16, torch.float16)


def grouped_gemm_checks(
    a: Tensor, b: Tensor, scale_a: Tensor, scale_b: Optional[Tensor], offsets: Tensor, rows: Optional[Tensor], output: Tensor,
) -> None:
    # Check shapes
    assert a.dim() == 2, f"Expected a to have 2 dimensions but got {a.dim() = } instead."
    assert b.dim() == 3 and a.size(1) == b.size(1), f"Expected {a.shape = } and {b.shape = } to be (rows, k) and (experts, k, n)."
    (a_rows, k), (experts, _, n) = a.shape, b.shape
    most = MAX_K if a.dtype == torch.int8 else 1 << 21
    assert k % 16 == 0 and 0 < k <= most, f"Expected {k = } to be a multiple of 16 from 16 to {most}"
    assert 1 <= n <= 1 << 21 and 1 <= experts <= _capi.MAX_EXPERTS, f"Expected {n = } to be between 1 and 2^21 and {experts = } up to {_capi.MAX_EXPERTS}"
    count = a_rows if rows is None else rows.numel()
    assert output.shape == (count, n), f"{output.shape} does not match with ({count}, {n})"
    assert scale_a.numel() in (1, a_rows), f"Expected scale_a to have 1 or {a_rows} elements but got {scale_a.shape}"
    assert scale_b is None or scale_b.shape in ((experts,), (experts, n)), f"Expected scale_b to be ({experts},) or ({experts}, {n}) but got {scale_b.shape}"
    assert offsets.shape == (experts + 1,), f"Expected offsets to be ({experts + 1},) but got {offsets.shape}"
    assert rows is None or rows.dim() == 1, f"Expected rows to have 1 dimension but got {rows.shape}"
    assert rows is None or a_rows * k < (1 << 31) - (1 << 22), f"Expected a to have less than 2^31 - 2^22 elements where rows picks from it: {a.shape = }"
    # Check dtypes
    assert a.dtype in (torch.float8_e4m3fn, torch.int8), f"Expected {a.dtype = } to be torch.float8_e4m3fn or torch.int8"
    assert b.dtype == a.dtype, f"Expected {b.dtype = } to be {a.dtype}"
    assert output.dtype in _OUT_DTYPES, f"Expected {output.dtype = } to be torch.bfloat16 or torch.float16"
    for name, t, dtype in (("scale_a", scale_a, torch.float32), ("scale_b", scale_b, torch.float32), ("offsets", offsets, torch.int32), ("rows", rows, torch.int32)):
        assert t is None or t.dtype == dtype, f"Expected {name} to be {dtype} but got {t.dtype}"
    # Check layouts
    for name, t in (("a", a), ("scale_a", scale_a), ("offsets", offsets), ("rows", rows), ("output", output)):
        assert t is None or t.is_contiguous(), f"Expected {name} to be contiguous but got {t.stride()}"
    assert b.stride(1) == 1, f"Expected b to have unit stride along k but got {b.stride() = }"
    assert n == 1 or (b.stride(2) >= k and b.stride(2) % 16 == 0 and b.stride(2) <= 1 << 21), \
        f"Expected b's columns to be a multiple of 16 bytes apart, at least {k}: {b.stride() = }"
    assert experts == 1 or b.stride(0) % 16 == 0, f"Expected b's experts to be a multiple of 16 bytes apart: {b.stride() = }"
    assert scale_b is None or scale_b.dim() == 1 or n == 1 or scale_b.stride(1) == 1, f"Expected scale_b to have unit stride along n but got {scale_b.stride()}"
    # Check devices
    device = a.device
    assert device.type == "cuda", f"Expected a.device to be of type cuda, but got {device.type = } instead."
    for name, t in (("b", b), ("scale_a", scale_a), ("scale_b", scale_b), ("offsets", offsets), ("rows", rows), ("output", output)):
        assert t is None or t.device == device, f"Expected {name} to be on {device} but got {t.device}"


def grouped_gemm(
    a: Tensor,
    b: Tensor,
    scale_a: Tensor,
    scale_b: Optional[Tensor],
    offsets: Tensor,
    rows: Optional[Tensor] = None,
    output: Optional[Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> Tensor:
    """Products of rows grouped by expert: row i of the result, offsets[e] <= i < offsets[e + 1], is scale_a[r] * scale_b[e] * (a[r] @ b[e]) with
    r = rows[i], or i without rows.  int8 sums are exact; float8_e4m3fn sums are the matrix cores' (a run of eight products is aligned to its largest and loses
    what is below 2^-13 of that, runs are added in fp32), as in every fp8 product here.  Scales in fp32, one rounding.
    Args:
        - a: a (rows, k) float8_e4m3fn or int8 tensor in row-major format, k a multiple of 16 (int8: up to 131056)
        - b: (experts, k, n) of a's dtype with unit stride along k (the `.transpose(1, 2)` of an (experts, n, k) weight); experts up to 512
        - scale_a: float32, one or one per row of a; scale_b: (experts, n), (experts,), or None: 1
        - offsets: (experts + 1,) int32, not decreasing, as `route_experts` gives them.  They stay on the device: no call waits for them, and a captured call
          may be replayed with others
        - rows: (count,) int32 or None: the row of a for each row of the result (`route_experts`' rows: a first projection picks the tokens' rows).  A
          number that is no row of a counts as a row of zeros (under a scale_b that is infinite or NaN the result there is zero or NaN)
        - output: a (count, n) tensor to write to, or None for a new one of out_dtype (bfloat16 or float16)
    Outputs:
        - (count, n); rows in front of offsets[0] and behind the last group's are not written.  Inference only: the result carries no gradient
    """
    if output is None and runs_now(a):
        out = _grouped_gemm_new(a, b, scale_a, scale_b, offsets, rows, out_dtype)
        if out is not None:  # one native operator; None: what is wrong, say the checks
            return out
    if output is None:
        output = torch.empty(size=(a.size(0) if rows is None else rows.numel(), b.size(-1)), dtype=out_dtype, device=a.device)
    grouped_gemm_checks(a, b, scale_a, scale_b, offsets, rows, output)
    _grouped_gemm(a, b, scale_a, scale_b, offsets, rows, output)
    return output
