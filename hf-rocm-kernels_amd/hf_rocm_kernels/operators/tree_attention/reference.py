"""Torch form of the attention, for callers who want to check the kernel.  The operators never call it."""
import math
from typing import Optional

import torch
from torch import Tensor


def reference_tree_attention(
    query: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None,
    mask: Optional[Tensor] = None, scale: Optional[float] = None, key_scale: Optional[Tensor] = None, value_scale: Optional[Tensor] = None,
    dtype: torch.dtype = torch.float64,
) -> Tensor:
    """`tree_attention` from its definition, one sequence and head at a time in `dtype`; what a row does not see takes no part in its sums
    (an infinity or a NaN there does not either).  Rows of no sequence are zero."""
    tokens, heads, head_dim = query.shape
    pages, page_size, kv_heads = key_cache.shape[:3]
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    seqs = page_table.size(0)
    edges = [b * (tokens // seqs) for b in range(seqs + 1)] if starts is None else starts.tolist()
    out = torch.zeros(query.shape, dtype=dtype, device=query.device)
    for b, length in enumerate(lengths.tolist()):
        first, last = edges[b], edges[b + 1]
        count, length = last - first, max(length, 0)
        token = torch.arange(min(length, page_table.size(1) * page_size), device=query.device)
        page = page_table[b].long()[token // page_size]
        here = (page >= 0) & (page < pages)
        place = token - (length - count)
        row = torch.arange(count, device=query.device)[:, None]
        if mask is None:
            sees = place <= row
        else:
            known = (place >= 0) & (place < min(count, mask.size(1)))
            sees = (place < 0).expand(count, -1).clone()
            sees[:, known] = mask[first:last].bool()[:, place[known]]
        sees = sees & here
        for h in range(heads):
            kv = h * kv_heads // heads

            def rows(cache, factor):
                # (each head's page by itself, as bytes where the type has no index kernel)
                one = cache[:, :, kv].contiguous()
                flat = one.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else one
                taken = flat[page.clamp(0, pages - 1), token % page_size]
                taken = taken.view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else taken
                return taken.to(dtype) * (1.0 if factor is None else factor.to(dtype).reshape(-1)[kv if factor.numel() > 1 else 0])

            k, v = rows(key_cache, key_scale), rows(value_cache, value_scale)
            score = (query[first:last, h].to(dtype) @ torch.where(here[:, None], k, 0.0).T) * scale
            score = torch.where(sees, score, -math.inf)
            weight = torch.softmax(score, dim=-1)
            weight = torch.where(sees.any(-1, keepdim=True), weight, 0.0)
            good = torch.isfinite(v)
            out[first:last, h] = weight @ torch.where(good, v, 0.0)
            for t in (~good).any(-1).nonzero().flatten().tolist():  # rare: one by one, to the rows that see it
                if bool(here[t]):
                    part = torch.where(good[t], torch.zeros((), dtype=dtype, device=v.device), v[t])
                    out[first:last, h] += torch.where(sees[:, t, None], weight[:, t, None] * part, 0.0)
    return out
