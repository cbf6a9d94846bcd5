"""Torch form of the grouped product, for callers who want to check the kernel.  The operator never calls it."""
from typing import Optional

import torch
from torch import Tensor


def _wide(codes: Tensor) -> Tensor:
    return codes.float().double()  # (not every device converts fp8 to 64 bits at once)


def reference_grouped_gemm(a: Tensor, b: Tensor, scale_a: Tensor, scale_b: Optional[Tensor], offsets: Tensor, rows: Optional[Tensor] = None) -> Tensor:
    """`grouped_gemm` in 64 bits, one expert at a time; rows of no group are zero, as are those whose number is no row of a."""
    count = a.size(0) if rows is None else rows.numel()
    out = torch.zeros((count, b.size(2)), dtype=torch.float64, device=a.device)
    edges = [min(max(x, 0), count) for x in offsets.tolist()]
    index = torch.arange(count, device=a.device) if rows is None else rows.long()
    known = (index >= 0) & (index < a.size(0))
    index = torch.where(known, index, 0)
    for e in range(b.size(0)):
        here = slice(edges[e], max(edges[e], edges[e + 1]))
        if edges[e] >= edges[e + 1]:
            continue
        wide = _wide(a) * scale_a.double().reshape(-1, 1)
        y = wide[index[here]] @ _wide(b[e])
        if scale_b is not None:
            y = y * scale_b[e].double().reshape(1, -1)
        out[here] = torch.where(known[here][:, None], y, 0.0)
    return out
