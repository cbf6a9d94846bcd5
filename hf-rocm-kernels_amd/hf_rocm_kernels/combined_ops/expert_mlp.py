from typing import Optional

import torch
from torch import Tensor

from hf_rocm_kernels import combine_experts, grouped_gemm, quantize_fp8, quantize_int8, route_experts, swiglu_dynamic


def expert_mlp_combined_ops(
    hidden: Tensor,
    logits: Tensor,
    top_k: int,
    gate_up_weight: Tensor,
    gate_up_scale: Optional[Tensor],
    down_weight: Tensor,
    down_scale: Optional[Tensor],
    residual: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    scoring: str = "softmax",
    renormalize: bool = True,
    factor: float = 1.0,
    mask: Optional[Tensor] = None,
) -> Tensor:
    """Decoder MLP sub-block of experts, six or eight launches on one stream: the normalised hidden states quantised per token, the router's choices, each expert's
    gate and up projection on its tokens, SwiGLU quantised per row, the down projections, and the weighted sum per token.

    - hidden: (tokens, hidden) 16-bit, as the layer's norm gives it; logits: (tokens, experts), the router's
    - gate_up_weight: (experts, 2 * inter, hidden) float8_e4m3fn or int8, an expert's gate rows in front of its up rows; down_weight: (experts, hidden, inter) of
      the same dtype; *_scale: float32, (experts, rows), (experts,) or None: 1
    - residual: (tokens, hidden) of hidden's dtype, added to the result (the residual stream, or a shared expert's result)
    - top_k, bias, scoring, renormalize, factor, mask: as `route_experts` takes them; a token of padding gets its residual, or zeros

    Nothing waits for the host: group sizes stay on the device, and a captured call can be replayed with other contents of the same tensors.
    Inference only.  Returns (tokens, hidden)."""
    int8 = gate_up_weight.dtype == torch.int8
    codes, scales = quantize_int8(hidden) if int8 else quantize_fp8(hidden)
    route = route_experts(logits, top_k, bias, scoring, renormalize, factor, mask)
    gate_up = grouped_gemm(codes, gate_up_weight.transpose(1, 2), scales, gate_up_scale, route.offsets, rows=route.rows, out_dtype=hidden.dtype)
    activated, scales = swiglu_dynamic(gate_up, dtype=gate_up_weight.dtype)
    down = grouped_gemm(activated, down_weight.transpose(1, 2), scales, down_scale, route.offsets, out_dtype=hidden.dtype)
    return combine_experts(down, route.weights, route.places, base=residual)
