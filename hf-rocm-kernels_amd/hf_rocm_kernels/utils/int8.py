import torch
from torch import Tensor

INT8_MAX = 127.0


def int8_quantize(x: Tensor, scale: Tensor) -> Tensor:
    """int8 codes rint(x / scale), ties to even, between -127 and 127 (the code -128 is not used: codes are symmetric).  A NaN becomes -127.
    `scale` may be a scalar tensor or broadcast against `x`."""
    return (x.float() / scale).round().nan_to_num(nan=-INT8_MAX).clamp(min=-INT8_MAX, max=INT8_MAX).to(torch.int8)


def int8_scale(x: Tensor, dim=None) -> Tensor:
    """scale = amax/127 over the whole tensor (dim=None) or per slice along `dim` (kept), never zero."""
    x = x.float().abs()
    amax = x.amax() if dim is None else x.amax(dim=dim, keepdim=True)
    return (amax / INT8_MAX).clamp_min(torch.finfo(torch.float32).tiny).to(torch.float32)
