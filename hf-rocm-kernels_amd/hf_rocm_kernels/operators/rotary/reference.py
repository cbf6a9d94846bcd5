"""Torch form of the rotation, for callers who want to check the kernel.  The operators never call it."""
import torch
from torch import Tensor


def reference_rotary(x: Tensor, positions: Tensor, frequencies: Tensor, interleaved: bool = False, magnitude: float = 1.0) -> Tensor:
    """`rotary` as a chain of torch calls: angles in float64, the rotation in the dtype that float32 and x's promote to, rounded to x's dtype once."""
    angles = positions.to(torch.float64)[:, None, None] * frequencies.to(torch.float64)
    work = torch.promote_types(x.dtype, torch.float32)
    cos, sin = (angles.cos() * magnitude).to(work), (angles.sin() * magnitude).to(work)
    rotated = 2 * frequencies.numel()
    head, rest = x[..., :rotated].to(work), x[..., rotated:]
    if interleaved:
        first, second = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((first * cos - second * sin, second * cos + first * sin), dim=-1).flatten(-2)
    else:
        first, second = head.chunk(2, dim=-1)
        turned = torch.cat((first * cos - second * sin, second * cos + first * sin), dim=-1)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)
