"""The attention sub-block: norm, projections, cache and attention as a layer runs them, against float64, over steps of several kinds."""
import math

import pytest
import torch

from hf_rocm_kernels import residual_rms, rotary, rotary_frequencies
from hf_rocm_kernels.combined_ops.llama_attention import llama_attention_combined_ops
from hf_rocm_kernels.combined_ops.llama_mlp import llama_mlp_combined_ops
from hf_rocm_kernels.layers.fp8_linear import apply_fp8_linear
from hf_rocm_kernels.utils.weight_format import pack_weight
from oracle import attention as oracle

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
HIDDEN, HEADS, KV_HEADS, HEAD_DIM, PAGE, PAGES, COLUMNS = 512, 8, 2, 64, 16, 24, 8


class Layer:
    def __init__(self, cache, dtype=torch.bfloat16, packed=False, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dtype = g, dtype
        rows = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        self.qkv = (torch.randn(rows, HIDDEN, generator=g) * 8).to(FP8).cuda()
        self.o = (torch.randn(HIDDEN, HEADS * HEAD_DIM, generator=g) * 8).to(FP8).cuda()
        self.qkv_scale = (torch.rand(rows, generator=g) * 0.004 + 0.004).cuda()
        self.o_scale = torch.tensor([0.005], device="cuda")
        self.norm = (1 + 0.1 * torch.randn(HIDDEN, generator=g)).to(dtype).cuda()
        self.qkv_input, self.o_input = torch.tensor([0.011], device="cuda"), torch.tensor([0.009], device="cuda")
        self.caches = [torch.full((PAGES, PAGE, KV_HEADS, HEAD_DIM), math.nan).to(cache or dtype).cuda() for _ in range(2)]
        self.scales = dict(key_scale=torch.tensor([0.02], device="cuda"), value_scale=torch.tensor([0.01, 0.02], device="cuda")) if cache else {}
        self.frequencies, self.magnitude = rotary_frequencies(HEAD_DIM, 500000.0)
        self.table = torch.randperm(PAGES, generator=g)[:2 * COLUMNS].view(2, COLUMNS).int()
        self.packed = packed

    def step(self, held, counts):
        """The arguments of a step that appends counts[b] tokens to sequence b, which holds held[b]."""
        at = [(b, t) for b in range(2) for t in range(held[b], held[b] + counts[b])]
        return dict(slots=torch.tensor([int(self.table[b, t // PAGE]) * PAGE + t % PAGE for b, t in at], dtype=torch.int32, device="cuda"),
                    positions=torch.tensor([t for _, t in at], dtype=torch.long, device="cuda"),
                    lengths=torch.tensor([h + n for h, n in zip(held, counts)], dtype=torch.int32, device="cuda"),
                    starts=torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device="cuda"))

    def rows(self, n):
        return [torch.randn(n, HIDDEN, generator=self.g).to(self.dtype).cuda() for _ in range(2)]

    def __call__(self, hidden, residual, step, mask=None, starts=True):
        step = step if starts else {k: v for k, v in step.items() if k != "starts"}
        return llama_attention_combined_ops(
            hidden, residual, self.norm, 1e-5, pack_weight(self.qkv) if self.packed else self.qkv, self.qkv_scale, self.qkv_input,
            pack_weight(self.o) if self.packed else self.o, self.o_scale, self.o_input, *self.caches, page_table=self.table.cuda(),
            frequencies=self.frequencies, mask=mask, magnitude=self.magnitude, **step, **self.scales)


@pytest.mark.parametrize("cache,dtype,packed", [(None, torch.bfloat16, False), (FP8, torch.bfloat16, True), (FP8, torch.float16, False)])
def test_steps_against_float64(cache, dtype, packed):
    """Prompts, a drafted tree, single tokens.  The norm, the projection and the rotation have tests of their own and are taken as they come; the cache is what the
    block has written.  Then attention within its tolerance, with its rounding to fp8, goes through the projection: by |weight| at most."""
    layer = Layer(cache, dtype, packed)
    held = [0, 0]
    for counts, tree in (([33, 70], False), ([5, 7], True), ([1, 1], False)):
        total, step = sum(counts), layer.step(held, counts)
        hidden, residual = layer.rows(total)
        mask = torch.rand(total, max(counts), generator=layer.g) < 0.5 if tree else None
        kept = residual.clone()
        out, residual_out = layer(hidden, residual, step, None if mask is None else mask.cuda(), starts=counts != [1, 1])
        assert residual_out is residual and out.dtype == dtype and out.shape == hidden.shape

        normalized, _ = residual_rms(input=hidden, residual=kept, weight=layer.norm, epsilon=1e-5, scale_tensor=layer.qkv_input)
        assert torch.equal(kept, residual)
        qkv = apply_fp8_linear(normalized, layer.qkv, layer.qkv_scale, layer.qkv_input, out_dtype=dtype).view(total, -1, HEAD_DIM)
        query = rotary(qkv[:, :HEADS], step["positions"], layer.frequencies)
        key = rotary(qkv[:, HEADS:HEADS + KV_HEADS], step["positions"], layer.frequencies)
        written = layer.caches[0].view(-1, KV_HEADS, HEAD_DIM)[step["slots"].long()].float()
        if cache:
            # the kernel divides before it rounds, here after a rounding to 16 bits: that half step, then one of fp8 around the value
            want = key.float() / 0.02
            assert ((written - want).abs() <= want.abs() * (oracle.half_step(FP8) + 2 * oracle.half_step(dtype)) + oracle.smallest_step(FP8)).all()
        else:
            assert torch.equal(written, key.float())

        scales = [None if s is None else s.cpu() for s in (layer.scales.get("key_scale"), layer.scales.get("value_scale"))]
        found = oracle.attention(query.cpu(), *[c.cpu() for c in layer.caches], layer.table, step["lengths"].cpu(), step["starts"].cpu(), mask,
                                 HEAD_DIM ** -0.5, *scales)
        o_input = float(layer.o_input)
        off = oracle.attention_tolerance(found, dtype, int(step["lengths"].max()), FP8, o_input).reshape(total, -1)
        attended = found[0].clamp(-448 * o_input, 448 * o_input).reshape(total, -1)
        weight = layer.o.cpu().double() * float(layer.o_scale)
        want = attended @ weight.T
        # sums of HEADS * HEAD_DIM products in fp32, two scales, the result's rounding
        size = (attended.abs() + off) @ weight.abs().T
        tol = off @ weight.abs().T + size * (HEADS * HEAD_DIM + 4) * 2.0 ** -24
        tol = tol + (want.abs() + tol) * oracle.half_step(dtype) * (1 + 2.0 ** -10) + oracle.smallest_step(dtype)
        assert float(((out.cpu().double() - want).abs() / tol).max()) <= 1.0
        held = [h + n for h, n in zip(held, counts)]


def test_captured_steps_and_padding():
    """A captured step of single tokens with two rows of padding, replayed for the next tokens, with eager work between; then the MLP's block on its result."""
    layer = Layer(None)
    step = layer.step([0, 0], [20, 37])
    layer(*layer.rows(57), step)
    held = [20, 37]
    hidden, residual = layer.rows(4)
    hidden[2:] = math.nan  # padding reaches nobody

    def padded(held):
        s = layer.step(held, [1, 1])
        return dict(slots=torch.cat([s["slots"], s["slots"].new_full((2,), -1)]), positions=torch.cat([s["positions"], s["positions"].new_zeros(2)]),
                    lengths=s["lengths"], starts=s["starts"])

    still = padded(held)
    table = layer.table.cuda()
    layer.table = table  # (its address is the captured one)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        layer(hidden, residual.clone(), still)  # eager on the stream of the capture: the projections' workspace
    torch.cuda.synchronize()
    residual_in = residual.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out, _ = layer(hidden, residual_in, still)
    up = (torch.randn(2 * 512, HIDDEN, device="cuda") * 4).to(FP8).t()
    down = (torch.randn(HIDDEN, 512, device="cuda") * 4).to(FP8).t()
    s = [torch.tensor([v], device="cuda") for v in (0.013, 0.0005, 0.01, 0.0004)]
    layer.table = layer.table.cpu()
    for _ in range(4):
        rows = layer.rows(4)
        hidden[:2] = rows[0][:2]
        residual_in.copy_(rows[1])
        for name, value in padded(held).items():
            still[name].copy_(value)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, cache = out.clone(), [c.clone() for c in layer.caches]
        after = rows[1].clone()
        want, _ = layer(hidden, after, padded(held))
        assert torch.isfinite(want[:2]).all() and torch.equal(got[:2], want[:2]) and torch.equal(after[:2], residual_in[:2])
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(cache, layer.caches))
        mlp, _ = llama_mlp_combined_ops(got[:2].clone(), residual_in[:2].clone(), layer.norm, 1e-5, up, s[0], s[1], down, s[2], s[3], fused=True)
        assert torch.isfinite(mlp).all()
        held = [h + 1 for h in held]


def test_no_tokens():
    layer = Layer(FP8)
    out, _ = layer(*layer.rows(0), layer.step([0, 0], [0, 0]))
    assert out.shape == (0, HIDDEN)


def test_refuses_projections_without_query_heads():
    layer = Layer(None)
    layer.qkv = layer.qkv[:2 * KV_HEADS * HEAD_DIM]
    layer.qkv_scale = layer.qkv_scale[:2 * KV_HEADS * HEAD_DIM]
    with pytest.raises(AssertionError, match="qkv_weight"):
        layer(*layer.rows(3), layer.step([0, 0], [1, 2]))
