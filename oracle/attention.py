"""Oracle of rotary positions, the paged cache's append and the attention over it, in float64 on the CPU.  Test infrastructure only (see
__init__.py).  No reference counterpart: the reference stops at the projections and the MLP block.

Every function also returns the sizes that a kernel's rounding errors scale with, so that tolerances are sums of half steps and not tuned."""
import math
from typing import Optional, Tuple

import torch
from torch import Tensor


def half_step(dtype: torch.dtype) -> float:
    """The most that rounding to `dtype` moves a normal value, relative to it."""
    return torch.finfo(dtype).eps / 2


def smallest_step(dtype: torch.dtype) -> float:
    """Half the distance of its subnormal values."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rotary(x: Tensor, positions: Tensor, frequencies: Tensor, interleaved: bool, magnitude: float = 1.0) -> Tuple[Tensor, Tensor]:
    """x (tokens, heads, head_dim) rotated, and per value the sum of the magnitudes it is made of (0 where copied)."""
    n = frequencies.numel()
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    for t in range(x.shape[0]):
        for j in range(n):
            a = float(positions[t]) * float(frequencies[j])
            c, s = magnitude * math.cos(a), magnitude * math.sin(a)
            i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
            u, v = x[t, :, i].double(), x[t, :, k].double()
            y[t, :, i], y[t, :, k] = u * c - v * s, v * c + u * s
            size[t, :, i] = size[t, :, k] = (u.abs() + v.abs()) * abs(magnitude)
    return y, size


def rotary_tolerance(want: Tensor, size: Tensor, dtype: torch.dtype) -> Tensor:
    """One rounding to `dtype`, and in fp32 in front of it: cosine and sine within 2^-22 (the turn as a float 2 pi 2^-26, the series' steps and the
    magnitude's the rest), two products and a sum of 2^-24 each: below 2^-21 of the sum of magnitudes."""
    return want.abs() * half_step(dtype) * (1 + 2.0 ** -10) + smallest_step(dtype) + size * 2.0 ** -21


def attention(query: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, lengths: Tensor, starts: Optional[Tensor],
              mask: Optional[Tensor], scale: float, key_scale: Optional[Tensor] = None, value_scale: Optional[Tensor] = None):
    """(result, sum_j p_j |v_j|, error bound of a score in fp32, largest |v|), rows of no sequence NaN; by the definition: what a row does not
    see takes no part, and one that sees nothing is zero."""
    tokens, heads, head_dim = query.shape
    pages, page_size, kv_heads = key_cache.shape[:3]
    seqs, columns = page_table.shape
    edges = starts.tolist() if starts is not None else [b * (tokens // max(seqs, 1)) for b in range(seqs + 1)]
    out = torch.full(query.shape, math.nan, dtype=torch.float64)
    spread, most = torch.zeros_like(out), torch.zeros_like(out)
    off = torch.zeros(query.shape[:2], dtype=torch.float64)
    for b in range(seqs):
        first, last = edges[b], edges[b + 1]
        length, n = max(int(lengths[b]), 0), last - first
        at = [t for t in range(min(length, columns * page_size)) if 0 <= int(page_table[b, t // page_size]) < pages]
        page = torch.tensor([int(page_table[b, t // page_size]) for t in at], dtype=torch.long)
        place = torch.tensor([t % page_size for t in at], dtype=torch.long)
        drafted = torch.tensor([t - (length - n) for t in at], dtype=torch.long)
        sees = torch.zeros((n, len(at)), dtype=torch.bool)
        for i in range(n):
            if mask is None:
                sees[i] = drafted <= i
            else:
                known = (drafted >= 0) & (drafted < min(n, mask.shape[1]))
                sees[i] = drafted < 0
                sees[i][known] = mask[first + i].bool()[drafted[known]]
        for h in range(kv_heads):
            ks = 1.0 if key_scale is None else float(key_scale.reshape(-1)[h if key_scale.numel() > 1 else 0])
            vs = 1.0 if value_scale is None else float(value_scale.reshape(-1)[h if value_scale.numel() > 1 else 0])
            k = key_cache[:, :, h].double()[page, place] * ks
            v = value_cache[:, :, h].double()[page, place] * vs
            for q_head in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                q = query[first:last, q_head].double()
                for i in range(n):
                    s = sees[i]
                    if not bool(s.any()):
                        out[first + i, q_head] = 0.0
                        continue
                    score = (k[s] @ q[i]) * scale
                    p = torch.softmax(score, 0)
                    out[first + i, q_head] = (p[:, None] * v[s]).sum(0)
                    good = torch.where(torch.isfinite(v[s]), v[s].abs(), 0.0)
                    spread[first + i, q_head] = p @ good
                    most[first + i, q_head] = good.amax(0)
                    # products in 32 bits, head_dim + 4 roundings; the difference to the largest score, its exponential
                    off[first + i, q_head] = float(((k[s].abs() @ q[i].abs()) * scale * ((head_dim + 4) * 2.0 ** -24)).max()
                                                   + (score.abs().max() * 4 + 4) * 2.0 ** -23)
    return out, spread, off, most


def attention_tolerance(found, dtype: torch.dtype, length: int, out_dtype: Optional[torch.dtype] = None, out_scale: float = 1.0) -> Tensor:
    """How far a kernel may be that keeps scores and sums in fp32 and rounds the weights to `dtype` and the result to `out_dtype`.

    A weight is off by half a step u and by the score's error e (relative), in the sum above the line and in the one below: 2 (u + e) of
    sum p |v|; sums of `length` terms in fp32 2^-24 each above and below; a weight below fp16's normal values by half its smallest step, 2^-25,
    where the largest weight, which is at most the sum, is 2^7 or more: length * 2^-32 * largest |v| (bf16 reaches as far down as fp32).  Then one rounding."""
    out, spread, off, most = found
    u = half_step(dtype)
    inner = 2 * (u + off[..., None]) * (1 + u) * spread + 2 * length * 2.0 ** -24 * spread
    inner = inner + (2 * length * smallest_step(dtype) * 2.0 ** -7 * most if dtype == torch.float16 else 0.0)
    if out_dtype is None:
        return inner + (out.abs() + inner) * half_step(dtype) * (1 + 2.0 ** -10) + smallest_step(dtype)
    return inner + (out.abs() + inner) * half_step(out_dtype) * (1 + 2.0 ** -10) + out_scale * smallest_step(out_dtype)
