"""Torch forms of the router and of the experts' sum, for callers who want to check the kernels.  The operators never call them."""
import math
from typing import Optional, Tuple

import torch
from torch import Tensor


def reference_route_experts(
    logits: Tensor, top_k: int, bias: Optional[Tensor] = None, scoring: str = "softmax", renormalize: bool = True, factor: float = 1.0,
    mask: Optional[Tensor] = None,
) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """`route_experts` from its definition in 64 bits, token by token: (weights, experts, places, rows, offsets)."""
    tokens, num_experts = logits.shape
    weights = torch.zeros((tokens, top_k), dtype=torch.float64)
    experts = torch.full((tokens, top_k), -1, dtype=torch.int32)
    for t in range(tokens):
        if mask is not None and not bool(mask[t]):
            continue
        x = logits[t].double().cpu()
        score = torch.sigmoid(x) if scoring == "sigmoid" else torch.zeros_like(x) if bool((x == -math.inf).all()) else torch.softmax(x, 0)
        key = x if bias is None else score + bias.double().cpu()
        key = torch.where((x > -math.inf) & (key > -math.inf), key, -math.inf)  # (NaN is not above anything)
        order = sorted((e for e in range(num_experts) if key[e] > -math.inf), key=lambda e: (-float(key[e]), e))[:top_k]
        for j, e in enumerate(order):
            experts[t, j], weights[t, j] = e, score[e]
        if renormalize and order:  # (by logarithms, which scores below 64 bits' range have too)
            logarithm = torch.nn.functional.logsigmoid(x) if scoring == "sigmoid" else torch.log_softmax(x, 0)
            weights[t, :len(order)] = torch.softmax(logarithm[order], 0)
        weights[t] *= factor
        if bool(torch.isnan(x).any() or torch.isnan(score).any()):
            weights[t] = math.nan
    flat = experts.reshape(-1).tolist()
    pairs = sorted((i for i in range(len(flat)) if flat[i] >= 0), key=lambda i: flat[i])  # (stable)
    places, rows = torch.full((len(flat),), -1, dtype=torch.int32), torch.full((len(flat),), -1, dtype=torch.int32)
    for place, i in enumerate(pairs):
        places[i], rows[place] = place, i // top_k
    offsets = torch.tensor([sum(1 for i in pairs if flat[i] < e) for e in range(num_experts + 1)], dtype=torch.int32)
    return weights, experts, places.reshape(tokens, top_k), rows, offsets


def reference_combine_experts(y: Tensor, weights: Tensor, places: Tensor, base: Optional[Tensor] = None) -> Tensor:
    """base + sum_j weights[:, j] * y[places[:, j]] in 64 bits; a place that is no row of y counts as zeros."""
    known = (places >= 0) & (places < y.size(0))
    out = torch.zeros((places.size(0), y.size(1)), dtype=torch.float64, device=y.device)
    for j in range(places.size(1)):
        row = torch.zeros_like(out)
        row[known[:, j]] = y[places[known[:, j], j].long()].double()
        out += weights[:, j, None].double() * row
    return out if base is None else out + base.double()
