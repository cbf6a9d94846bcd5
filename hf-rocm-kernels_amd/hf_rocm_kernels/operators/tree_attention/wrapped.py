import math
from typing import Optional

import torch
from torch import Tensor

from ...utils.dispatch import runs_now
from ..append_kv.wrapped import cache_checks, scale_checks
from ..rotary.wrapped import heads_checks
from .binding import _tree_attention

_tree_attention_new = torch.ops._HFRK_C.tree_attention_new.default
MAX_HEAD_DIM = 256


def tree_attention_checks(
    query: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, lengths: Tensor, starts: Optional[Tensor], mask: Optional[Tensor],
    scale: float, key_scale: Optional[Tensor], value_scale: Optional[Tensor], out_scale: Optional[Tensor], output: Tensor,
) -> None:
    heads_checks("query", query)
    tokens, heads, head_dim = query.shape
    device = query.device
    assert key_cache.dim() == 4, f"Expected key_cache to have 4 dimensions (pages, page_size, kv_heads, head_dim) but got {key_cache.shape}"
    kv_heads, page_size = key_cache.size(2), key_cache.size(1)
    cache_checks(key_cache, value_cache, kv_heads, head_dim, query.dtype, device)
    fp8 = key_cache.dtype == torch.float8_e4m3fn
    assert heads >= 1 and kv_heads >= 1 and heads % kv_heads == 0, f"Expected {heads = } to be a multiple of {kv_heads = }"
    multiple = 16 if fp8 or head_dim > 128 else 8
    assert 16 <= head_dim <= MAX_HEAD_DIM and head_dim % multiple == 0, \
        f"Expected {head_dim = } to be a multiple of {multiple} from 16 to {MAX_HEAD_DIM}"
    assert page_size % 8 == 0, f"Expected {page_size = } to be a multiple of 8"
    assert page_table.dim() == 2 and page_table.dtype == torch.int32, f"Expected page_table to be (seqs, columns) int32 but got {page_table.shape} {page_table.dtype}"
    assert page_table.size(1) <= 1 or page_table.stride(1) == 1, f"Expected page_table to have unit stride along its rows but got {page_table.stride()}"
    seqs = page_table.size(0)
    assert page_table.size(1) * page_size <= 1 << 27, f"Expected at most 2^27 places in a row of page_table: {page_table.shape = }, {page_size = }"
    assert tokens * heads <= 1 << 28, f"Expected at most 2^28 query heads in a call: {query.shape = }"
    assert tokens == 0 or (key_cache.size(0) >= 1 and page_table.size(1) >= 1), "Expected a page and a column of page_table at least"
    for name, x, count in (("lengths", lengths, seqs), ("starts", starts, seqs + 1)):
        if x is not None:
            assert x.shape == (count,) and x.dtype == torch.int32 and x.is_contiguous(), f"Expected {name} to be {count} int32 values but got {x.shape} {x.dtype}"
            assert x.device == device, f"Expected {name} to be on {device} but got {x.device}"
    if starts is None:
        assert (tokens % seqs if seqs else tokens) == 0, f"Expected starts, or the same number of tokens for each of {seqs} sequences: {query.shape = }"
    if mask is not None:
        assert mask.dim() == 2 and mask.size(0) == tokens and mask.dtype in (torch.bool, torch.uint8), \
            f"Expected mask to be ({tokens}, drafted) bool or uint8 but got {mask.shape} {mask.dtype}"
        assert mask.size(1) <= 1 or mask.stride(1) == 1, f"Expected mask to have unit stride along its rows but got {mask.stride()}"
        assert mask.device == device, f"Expected mask to be on {device} but got {mask.device}"
    assert scale > 0, f"Expected {scale = } to be > 0"
    scale_checks(key_scale, value_scale, kv_heads, key_cache)
    if out_scale is not None:
        assert out_scale.numel() == 1 and out_scale.dtype == torch.float32 and out_scale.device == device, "Expected out_scale to be one float32 on the query's device"
    wanted = query.dtype if out_scale is None else torch.float8_e4m3fn
    assert output.shape == query.shape and output.dtype == wanted, f"Expected output to be {query.shape} {wanted} but got {output.shape} {output.dtype}"
    assert output.stride(2) == 1, f"Expected output to have unit stride along head_dim but got {output.stride()}"
    assert output.device == device and page_table.device == device, f"Expected output and page_table to be on {device}"
    assert device.type == "cuda", f"Expected query.device to be of type cuda, but got {device.type = } instead."


def tree_attention(
    query: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    page_table: Tensor,
    lengths: Tensor,
    starts: Optional[Tensor] = None,
    mask: Optional[Tensor] = None,
    scale: Optional[float] = None,
    key_scale: Optional[Tensor] = None,
    value_scale: Optional[Tensor] = None,
    out_scale: Optional[Tensor] = None,
    output: Optional[Tensor] = None,
) -> Tensor:
    """Attention of a step's queries over a paged cache that already holds the step's own keys and values (`append_kv`): one token a sequence
    (decode), a chain of tokens (a prompt's chunk, a linear draft) or a tree of drafted tokens.
    Args:
        - query: a 16-bit (bfloat16 or float16) tensor of shape (tokens, heads, head_dim), heads a multiple of the cache's kv_heads
        - key_cache, value_cache: as `append_kv` writes them, of the query's dtype or float8_e4m3fn; page_size a multiple of 8, head_dim one from 16 on
            (of 16 with float8_e4m3fn and above 128) up to 256
        - page_table: (seqs, columns) int32: a sequence's pages in order.  Entries that are no page (-1) hold nothing that is seen
        - lengths: (seqs, ) int32, the cached tokens of each sequence, those of this step included: they are its last ones
        - starts: (seqs + 1, ) int32: sequence b's tokens are rows starts[b] .. starts[b+1] of query; None: the same number each
        - mask: (tokens, drafted) bool or uint8: whether a token sees the j-th token of its sequence's step, as many columns as the longest step
            has (columns that are missing are not seen); None: a chain, each sees itself and those in front.  Tokens in front of the step are
            seen by all of it
        - scale: the scores' factor, 1/sqrt(head_dim) when None
        - key_scale, value_scale: the positive scales of float8_e4m3fn caches, as in `append_kv`
        - out_scale: one float32: the result is divided by it and converted to float8_e4m3fn (saturating, NaN kept), as the projection behind it takes it
        - output: a tensor to write to; None: a new one
    Outputs:
        - (tokens, heads, head_dim) of the query's dtype, or float8_e4m3fn with out_scale.  A token that sees nothing gets zeros, one whose scores
          are all minus infinity NaN; rows behind the last sequence's are not written.  Inference only: the result carries no gradient
    Each call takes a workspace from torch's allocator for parts of rows: up to about 128 MiB and 16 bytes a token and query head of a group.
    A batch of some thousand short sequences is slow, as every workgroup looks at all of them; one of 65536 with more than about 15 kv_heads is refused.
    Lengths, starts and page_table stay on the device: no call waits for them, and a captured call may be replayed with others.  The result does not depend
    on other streams' calls (each has a workspace of its own), but how a sequence's tokens are split, and with it the last bits, depends on all lengths.
    """
    if output is None and runs_now(query):
        output = _tree_attention_new(query, key_cache, value_cache, page_table, lengths, starts, mask, scale, key_scale, value_scale, out_scale)
        if output is not None:  # one native operator; None: what is wrong, say the checks
            return output
    if scale is None:
        scale = 1.0 / math.sqrt(query.size(-1))
    if output is None:
        output = torch.empty(size=query.shape, dtype=query.dtype if out_scale is None else torch.float8_e4m3fn, device=query.device)
    tree_attention_checks(query, key_cache, value_cache, page_table, lengths, starts, mask, scale, key_scale, value_scale, out_scale, output)
    _tree_attention(query, key_cache, value_cache, page_table, lengths, starts, mask, scale, key_scale, value_scale, out_scale, output)
    return output
