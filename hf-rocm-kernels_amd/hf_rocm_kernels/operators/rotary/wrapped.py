from typing import Optional

import torch
from torch import Tensor

from ...utils.dispatch import runs_now
from .binding import _rotary

_rotary_new = torch.ops._HFRK_C.rotary_new.default
_IO_DTYPES = (torch.bfloat16, torch.float16)
MAX_HEAD_DIM = 1024


def rotation_checks(tokens: int, head_dim: int, positions: Tensor, frequencies: Tensor, device: torch.device) -> None:
    assert positions.shape == (tokens,), f"Expected {positions.shape = } to be {(tokens,)}"
    assert positions.dtype in (torch.int32, torch.int64), f"Expected {positions.dtype = } to be torch.int32 or torch.int64"
    assert frequencies.dim() == 1 and 2 * frequencies.numel() <= head_dim, \
        f"Expected at most {head_dim // 2} frequencies but got {frequencies.shape = }"
    assert frequencies.dtype in (torch.float32, torch.float64), f"Expected {frequencies.dtype = } to be torch.float32 or torch.float64"
    assert positions.is_contiguous() and frequencies.is_contiguous(), "Expected positions and frequencies to be contiguous"
    assert positions.device == device, f"Expected {positions.device = } to be {device}"
    assert frequencies.device == device, f"Expected {frequencies.device = } to be {device}"


def heads_checks(name: str, x: Tensor) -> None:
    assert x.dim() == 3, f"Expected {name} to have 3 dimensions (tokens, heads, head_dim) but got {x.shape}"
    assert x.dtype in _IO_DTYPES, f"Expected {name} to be torch.bfloat16 or torch.float16 but got {x.dtype}"
    assert x.size(2) <= 1 or x.stride(2) == 1, f"Expected {name} to have unit stride along head_dim but got {x.stride()}"
    assert 1 <= x.size(2) <= MAX_HEAD_DIM, f"Expected {name} to have heads of 1 to {MAX_HEAD_DIM} values but got {x.shape}"


def rotary_checks(x: Tensor, positions: Tensor, frequencies: Tensor, output: Tensor) -> None:
    heads_checks("x", x)
    assert output.shape == x.shape and output.dtype == x.dtype, f"Expected output like x but got {output.shape = } {output.dtype = }"
    assert output.size(2) <= 1 or output.stride(2) == 1, f"Expected output to have unit stride along head_dim but got {output.stride() = }"
    rotation_checks(x.size(0), x.size(2), positions, frequencies, x.device)
    assert output.device == x.device, f"Expected {output.device = } to be {x.device}"
    assert x.device.type == "cuda", f"Expected x.device to be of type cuda, but got {x.device.type = } instead."


def rotary(
    x: Tensor,
    positions: Tensor,
    frequencies: Tensor,
    interleaved: bool = False,
    magnitude: float = 1.0,
    output: Optional[Tensor] = None,
) -> Tensor:
    """Rotary positions on the heads of a step: each pair of a head's first 2 * len(frequencies) values is turned by position * frequency.
    Args:
        - x: a 16-bit (bfloat16 or float16) tensor of shape (tokens, heads, head_dim), unit stride along head_dim, any strides
            else: the query and key heads of a projection's output are one call when they lie side by side
        - positions: (tokens, ) int32 or int64
        - frequencies: radians per position, float64 or float32, one per pair (`rotary_frequencies`); fewer than head_dim / 2
            leave the end of each head as it is
        - interleaved: pairs are neighbours (2j, 2j+1) instead of (j, j + len(frequencies))
        - magnitude: a factor on the turned values (`rotary_frequencies` gives it)
        - output: a tensor like x to write to, x itself to rotate in place; None: a new contiguous one
    Angles are formed in 64 bits, the rotation in 32, rounded once.  Inference only: the result carries no gradient.
    """
    if output is None:
        if runs_now(x):
            output = _rotary_new(x, positions, frequencies, magnitude, interleaved)  # one native operator; None: what is wrong, say the checks
            if output is not None:
                return output
        output = torch.empty(size=x.shape, dtype=x.dtype, device=x.device)
    rotary_checks(x, positions, frequencies, output)
    _rotary(x, positions, frequencies, magnitude, interleaved, output)
    return output
