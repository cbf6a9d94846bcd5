from typing import NamedTuple, Optional

import torch
from torch import Tensor

from ... import _capi
from ...utils.dispatch import runs_now
from .binding import _combine_experts, _route_experts

_route_experts_new = torch.ops._HFRK_C.route_experts_new.default
_combine_experts_new = torch.ops._HFRK_C.combine_experts_new.default
_SCORINGS = ("softmax", "sigmoid")
_LOGITS = (torch.bfloat16, torch.float16, torch.float32)
_IO_DTYPES = (torch.bfloat16, torch.float16)


class ExpertRoute(NamedTuple):
    """Which experts the tokens go to, and the (token, choice) pairs in the experts' order."""
    weights: Tensor   # (tokens, top_k) float32
    experts: Tensor   # (tokens, top_k) int32, -1: none
    places: Tensor    # (tokens, top_k) int32: where each pair is in the experts' order, -1: nowhere
    rows: Tensor      # (tokens * top_k,) int32: the token of each pair in that order, -1 behind the last one
    offsets: Tensor   # (num_experts + 1,) int32: expert e has the pairs offsets[e] .. offsets[e + 1]


def route_experts_checks(logits: Tensor, top_k: int, bias: Optional[Tensor], scoring: str, mask: Optional[Tensor]) -> None:
    assert logits.dim() == 2, f"Expected logits to have 2 dimensions but got {logits.shape}"
    tokens, num_experts = logits.shape
    assert logits.dtype in _LOGITS, f"Expected {logits.dtype = } to be one of {_LOGITS}"
    assert 1 <= num_experts <= _capi.MAX_EXPERTS, f"Expected {num_experts = } to be between 1 and {_capi.MAX_EXPERTS}"
    assert 1 <= top_k <= min(num_experts, _capi.MAX_TOP), f"Expected {top_k = } to be between 1 and {num_experts = }, {_capi.MAX_TOP} at most"
    assert tokens <= 1 << 24 and tokens * top_k <= 1 << 28, f"Expected at most 2^24 tokens and 2^28 pairs: {tokens = }, {top_k = }"
    assert num_experts == 1 or logits.stride(1) == 1, f"Expected logits to have unit stride along the experts but got {logits.stride()}"
    assert scoring in _SCORINGS, f"Expected {scoring = } to be one of {_SCORINGS}"
    if bias is not None:
        assert bias.shape == (num_experts,) and bias.dtype == torch.float32 and bias.is_contiguous(), \
            f"Expected bias to be {num_experts} contiguous float32 values but got {bias.shape} {bias.dtype}"
    if mask is not None:
        assert mask.shape == (tokens,) and mask.dtype in (torch.bool, torch.uint8) and mask.is_contiguous(), \
            f"Expected mask to be {tokens} contiguous bool or uint8 values but got {mask.shape} {mask.dtype}"
    device = logits.device
    assert device.type == "cuda", f"Expected logits.device to be of type cuda, but got {device.type = } instead."
    for name, t in (("bias", bias), ("mask", mask)):
        assert t is None or t.device == device, f"Expected {name} to be on {device} but got {t.device}"


def route_experts(
    logits: Tensor,
    top_k: int,
    bias: Optional[Tensor] = None,
    scoring: str = "softmax",
    renormalize: bool = True,
    factor: float = 1.0,
    mask: Optional[Tensor] = None,
) -> ExpertRoute:
    """Which experts each token goes to, with what weight, and the tokens in the experts' order, as `grouped_gemm` and `combine_experts` take them.
    Args:
        - logits: (tokens, num_experts) bfloat16, float16 or float32, unit stride along the experts; up to 512 experts
        - top_k: experts per token, up to 32
        - bias: (num_experts,) float32 that is added to the scores for the choice, not to the weights; None: the largest logits are chosen.  Of equals the lowest
          index comes first.  The choice is the one that sums in 64 bits give
        - scoring: "softmax" over a token's logits, or "sigmoid" of each
        - renormalize: divide a token's weights by their sum.  It is taken of the scores as they are, those below fp32's range among them
        - factor: what the weights are multiplied by at the end
        - mask: (tokens,) bool or uint8: tokens that are 0 are padding and go nowhere
    Outputs:
        - an `ExpertRoute`.  An expert whose logit (or sum with the bias) is minus infinity or NaN is never chosen; where too few are left the expert is -1
          and the weight 0.  A NaN among a token's logits, or with "softmax" a plus infinity, makes its weights NaN
    Equal calls give equal bits.  Inference only: the weights carry no gradient.
    """
    if scoring in _SCORINGS and runs_now(logits):
        found = _route_experts_new(logits, top_k, bias, scoring == "sigmoid", renormalize, factor, mask)
        if found[0] is not None:  # one native operator; None: what is wrong, say the checks
            return ExpertRoute(*found)
    route_experts_checks(logits, top_k, bias, scoring, mask)
    tokens, num_experts = logits.shape

    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=logits.device)

    route = ExpertRoute(torch.empty((tokens, top_k), dtype=torch.float32, device=logits.device), ints(tokens, top_k), ints(tokens, top_k), ints(tokens * top_k),
                        ints(num_experts + 1))
    _route_experts(logits, top_k, bias, scoring == "sigmoid", renormalize, factor, mask, *route)
    return route


def combine_experts_checks(y: Tensor, weights: Tensor, places: Tensor, base: Optional[Tensor], output: Tensor) -> None:
    assert y.dim() == 2 and y.size(1) >= 1 and y.size(1) <= 1 << 21, f"Expected y to be (rows, cols), cols up to 2^21, but got {y.shape}"
    assert y.dtype in _IO_DTYPES, f"Expected {y.dtype = } to be torch.bfloat16 or torch.float16"
    assert places.dim() == 2 and places.dtype == torch.int32, f"Expected places to be (tokens, top_k) int32 but got {places.shape} {places.dtype}"
    assert 1 <= places.size(1) <= _capi.MAX_TOP, f"Expected {places.size(1) = } to be between 1 and {_capi.MAX_TOP}"
    assert weights.shape == places.shape and weights.dtype == torch.float32, f"Expected weights to be {places.shape} float32 but got {weights.shape} {weights.dtype}"
    shape = (places.size(0), y.size(1))
    assert places.size(0) < 1 << 24, f"Expected less than 2^24 tokens: {places.shape = }"
    assert base is None or (base.shape == shape and base.dtype == y.dtype), f"Expected base to be {shape} {y.dtype} but got {base.shape} {base.dtype}"
    assert output.shape == shape and output.dtype == y.dtype, f"Expected output to be {shape} {y.dtype} but got {output.shape} {output.dtype}"
    device = y.device
    assert device.type == "cuda", f"Expected y.device to be of type cuda, but got {device.type = } instead."
    for name, t in (("y", y), ("weights", weights), ("places", places), ("base", base), ("output", output)):
        assert t is None or t.is_contiguous(), f"Expected {name} to be contiguous but got {t.stride()}"
        assert t is None or t.device == device, f"Expected {name} to be on {device} but got {t.device}"


def combine_experts(y: Tensor, weights: Tensor, places: Tensor, base: Optional[Tensor] = None, output: Optional[Tensor] = None) -> Tensor:
    """base[t] + sum_j weights[t, j] * y[places[t, j]]: the rows that a token's experts made, weighted, in fp32, rounded once.
    Args:
        - y: (rows, cols) bfloat16 or float16: the second projection's rows, in the experts' order
        - weights, places: (tokens, top_k) float32 and int32, as `route_experts` gives them.  A place that is no row of y (-1) counts as a row of zeros
        - base: an addend (tokens, cols) of y's dtype (the residual stream, a shared expert's result) or None
        - output: a tensor to write to (it may be base), or None for a new one
    Equal calls give equal bits: a token's choices are added in their order.  Inference only: the result carries no gradient.
    """
    if output is None and runs_now(y):
        out = _combine_experts_new(y, weights, places, base)
        if out is not None:  # one native operator; None: what is wrong, say the checks
            return out
    if output is None:
        output = torch.empty(size=(places.size(0), y.size(-1)), dtype=y.dtype, device=y.device)
    combine_experts_checks(y, weights, places, base, output)
    _combine_experts(y, weights, places, base, output)
    return output
