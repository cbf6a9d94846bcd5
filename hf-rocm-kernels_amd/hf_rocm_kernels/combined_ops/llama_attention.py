from typing import Optional, Tuple

import torch
from torch import Tensor

from hf_rocm_kernels import append_kv, residual_rms, tree_attention

from ..layers.fp8_linear import Weight, apply_fp8_linear


def llama_attention_combined_ops(
    hidden: Tensor,
    residual: Tensor,
    rms_weight: Tensor,
    rms_epsilon: float,
    qkv_weight: Weight,
    qkv_weight_scale: Optional[Tensor],
    qkv_input_scale: Tensor,
    o_weight: Weight,
    o_weight_scale: Optional[Tensor],
    o_input_scale: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    slots: Tensor,
    positions: Tensor,
    frequencies: Tensor,
    page_table: Tensor,
    lengths: Tensor,
    starts: Optional[Tensor] = None,
    mask: Optional[Tensor] = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
    scale: Optional[float] = None,
    key_scale: Optional[Tensor] = None,
    value_scale: Optional[Tensor] = None,
) -> Tuple[Tensor, Tensor]:
    """Decoder attention sub-block over a paged cache, five launches on one stream (six where the cache is split between workgroups):
    residual RMSNorm -> fp8, qkv GEMM, keys rotated and appended with the values (the queries rotated along with them), attention over the cache -> fp8,
    output GEMM.  What it returns is what `llama_mlp_combined_ops` takes next.

    - hidden, residual: (tokens, hidden) 16-bit; residual <- hidden + residual in place
    - qkv_weight: ((heads + 2 * kv_heads) * head_dim, hidden) float8_e4m3fn, rows of the query heads, the key heads, the value heads, or its
      PackedWeight; o_weight: (hidden, heads * head_dim); *_weight_scale: one float32 or one per row, or None for a PackedWeight that carries its own
    - qkv_input_scale, o_input_scale: one float32: the quantisation scales of the two GEMMs' activations
    - key_cache, value_cache, slots, key_scale, value_scale, positions, frequencies, interleaved, magnitude: as `append_kv` takes them; modified in place
    - page_table, lengths (this step's tokens included), starts, mask, scale: as `tree_attention` takes them

    Rows of padding (a negative slot, behind starts' last) take no part in other rows; theirs of the first output hold nothing.
    Nothing waits for the host, and a captured call can be replayed with other positions, slots, lengths, pages and masks in the same tensors.  Run one eager
    call on the stream of the capture first: the projections' workspace is the stream's.
    Inference only.  Returns (attn_output, residual)."""
    tokens = hidden.size(0)
    kv_heads, head_dim = key_cache.size(2), key_cache.size(3)
    normalized, residual = residual_rms(input=hidden, residual=residual, weight=rms_weight, epsilon=rms_epsilon, scale_tensor=qkv_input_scale)
    qkv = apply_fp8_linear(normalized, qkv_weight, qkv_weight_scale, qkv_input_scale, out_dtype=hidden.dtype)
    heads = qkv.size(1) // head_dim - 2 * kv_heads
    assert qkv.size(1) % head_dim == 0 and heads > 0, f"Expected qkv_weight to have rows of more than {2 * kv_heads} heads of {head_dim} but got {qkv.size(1)}"
    query, key, value = qkv.view(tokens, heads + 2 * kv_heads, head_dim).split((heads, kv_heads, kv_heads), dim=1)
    query = append_kv(key, value, key_cache, value_cache, slots, positions, frequencies, interleaved, magnitude, query=query, key_scale=key_scale,
                      value_scale=value_scale)
    attended = tree_attention(query, key_cache, value_cache, page_table, lengths, starts, mask, scale, key_scale, value_scale, out_scale=o_input_scale)
    attn_output = apply_fp8_linear(attended.view(tokens, heads * head_dim), o_weight, o_weight_scale, o_input_scale, out_dtype=hidden.dtype)
    return attn_output, residual
