"""Linear layers on int8 weights, beside the fp8 ones: the same calls, for checkpoints in 8-bit integers (one scale per output channel, activations
quantised per token or with one static scale).

A call runs as one quantisation kernel (skipped where the caller holds int8 activations and their scales, e.g. from `swiglu_dynamic(dtype=torch.int8)`) and one
product with the scales, the bias or the residual in its epilogue.
"""
from typing import Optional

import torch
from torch import Tensor

from ..operators.int8_gemm import int8_gemm
from ..operators.quantize import quantize_int8
from ..utils.dispatch import runs_now
from ..utils.int8 import int8_quantize, int8_scale

_int8_linear = torch.ops._HFRK_C.int8_linear.default


def apply_int8_linear(
    input: Tensor,
    weight: Tensor,
    weight_scale: Optional[Tensor],
    input_scale: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    residual: Optional[Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> Tensor:
    """y = input @ dequant(weight).T (+ bias) (+ residual), computed on int8 codes with exact sums.

    - input: (..., k) float16/bfloat16 activations, quantised here -- with `input_scale` (one float32: static) or, when it is None, dynamically per
      token -- or an int8 tensor already quantised, `input_scale` then being its scale(s): one float32 or one per token
    - weight: (n, k) int8 row-major; weight_scale: one float32 or one per output channel, None: 1
    - bias: (n,) in the output dtype (any shape and dtype that broadcasts to the output is taken); residual: (..., n) in the output dtype, added in the
      product's epilogue (fp32 sum, one rounding).  Given both, the bias is added to the residual first (one 16-bit add).
    - out_dtype: float16/bfloat16; defaults to the input's (bfloat16 for an int8 input)
    Inference only: the result carries no gradient.
    """
    if runs_now(input):  # usual calls run as one native operator; None: not one of those
        out = _int8_linear(input, weight, weight_scale, input_scale, bias, residual, out_dtype)
        if out is not None:
            return out
    k, n = input.shape[-1], weight.size(0)
    lead = input.shape[:-1]
    x = input.reshape(-1, k)
    if x.dtype == torch.int8:
        assert input_scale is not None, "an int8 input needs its scale(s)"
        codes, scales = x.contiguous(), input_scale.reshape(-1)
        out_dtype = out_dtype or torch.bfloat16
    else:
        out_dtype = out_dtype or x.dtype
        codes, scales = quantize_int8(x.contiguous(), input_scale)
        scales = scales.reshape(-1)
    m = codes.size(0)
    if scales.numel() != 1:
        scales = scales[:m]  # a buffer of scales may be longer than the batch
    base = None
    if residual is not None:
        base = residual.reshape(m, n)
        if bias is not None:
            base = base + bias
        base = base.contiguous()
    elif bias is not None:
        base = bias.to(out_dtype)
        base = base.contiguous() if base.shape == (n,) else base.expand(*lead, n).reshape(m, n).contiguous()
    out = torch.empty((m, n), dtype=out_dtype, device=codes.device)
    int8_gemm(codes, weight.t(), scales, None if weight_scale is None else weight_scale.reshape(-1), base, output=out)
    return out.reshape(*lead, n)


class Int8Linear(torch.nn.Module):
    """nn.Linear with an int8 weight: per-output-channel (default) or per-tensor weight scale, dynamic per-token or static activation scale.  Inference
    only.

    The tensors are registered buffers (`weight`, `weight_scale`, `bias`, `input_scale`), so the layer moves with `.to()` and round-trips through
    `state_dict()` / `load_state_dict()`."""

    def __init__(self, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor] = None, input_scale: Optional[Tensor] = None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)
        self.register_buffer("input_scale", input_scale)

    def _apply(self, fn, *args, **kwargs):
        """Device moves reach every buffer; dtype casts (`.half()`, `.to(torch.bfloat16)`) reach the bias only: the float32 scales keep their dtype."""
        before = {name: getattr(self, name) for name in ("weight", "weight_scale", "input_scale")}
        module = super()._apply(fn, *args, **kwargs)
        for name, old in before.items():
            new = getattr(self, name)
            if old is not None and new is not None and new.dtype != old.dtype:
                self._buffers[name] = old.to(new.device)
        return module

    @classmethod
    def from_float(cls, linear: torch.nn.Linear, per_channel: bool = True, input_scale: Optional[Tensor] = None) -> "Int8Linear":
        """Quantise an nn.Linear's weight (scale = amax/127 per output channel or per tensor)."""
        w = linear.weight.detach()
        scale = int8_scale(w, dim=1 if per_channel else None)
        bias = None if linear.bias is None else linear.bias.detach().clone()
        return cls(int8_quantize(w, scale), scale.reshape(-1).contiguous(), bias, input_scale)

    def forward(self, input: Tensor, input_scale: Optional[Tensor] = None, residual: Optional[Tensor] = None) -> Tensor:
        """`input` 16-bit (quantised here) or int8 with `input_scale`; `residual` is added in the product's epilogue."""
        return apply_int8_linear(input, self.weight, self.weight_scale, self.input_scale if input_scale is None else input_scale, self.bias, residual)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
