"""Products by expert, int8 products, router and sum on the host: the C entry points refuse what the kernels do not take before they touch a device, the
wrappers trace, and the plain forms agree with each other."""
import ctypes

import pytest
import torch
from torch._subclasses import FakeTensorMode

import hf_rocm_kernels
from hf_rocm_kernels import _capi
from hf_rocm_kernels.combined_ops.expert_mlp import expert_mlp_combined_ops
from hf_rocm_kernels.layers import Int8Linear, apply_int8_linear
from hf_rocm_kernels.operators.experts import reference_combine_experts, reference_route_experts
from hf_rocm_kernels.operators.grouped_gemm import reference_grouped_gemm
from hf_rocm_kernels.utils.int8 import int8_quantize, int8_scale

LIB = _capi.load()
P = 1 << 20  # an address that is never read: every call here is refused, or has nothing to do
FP8, INT8 = torch.float8_e4m3fn, torch.int8


def _grouped(**changes):
    args = dict(a=P, rows=P, b=P, expert_stride=64 * 32, output=P, scale_a=P, scale_b=P, scale_b_expert_stride=32, offsets=P, scale_a_stride=1, scale_b_stride=1,
                b_stride=64, count=10, a_rows=5, experts=4, n=32, k=64, type=_capi.FP8_E4M3FN, dtype=_capi.BF16)
    args.update(changes)
    return LIB.hfrk_grouped_gemm(ctypes.byref(_capi.GroupedArgs(**args)), None)


@pytest.mark.parametrize("changes,status", [
    ({"a": None}, _capi.BAD_SHAPE), ({"b": None}, _capi.BAD_SHAPE), ({"output": None}, _capi.BAD_SHAPE), ({"scale_a": None}, _capi.BAD_SHAPE),
    ({"offsets": None}, _capi.BAD_SHAPE), ({"experts": 0}, _capi.BAD_SHAPE), ({"experts": 513}, _capi.BAD_SHAPE), ({"n": 0}, _capi.BAD_SHAPE),
    ({"n": (1 << 21) + 1}, _capi.BAD_SHAPE), ({"k": 0}, _capi.BAD_SHAPE), ({"k": 24, "b_stride": 32}, _capi.K_NOT_DIVISIBLE_BY_WARPTILE_K), ({"count": -1}, _capi.BAD_SHAPE),
    ({"type": _capi.BF16}, _capi.BAD_DTYPE), ({"dtype": _capi.FP8_E4M3FN}, _capi.BAD_DTYPE), ({"dtype": _capi.FP32}, _capi.BAD_DTYPE), ({"b_stride": 48}, _capi.BAD_SHAPE),
    ({"b_stride": 72}, _capi.BAD_ALIGNMENT), ({"b_stride": 1 << 22}, _capi.BAD_SHAPE), ({"expert_stride": -64}, _capi.BAD_SHAPE),
    ({"expert_stride": 8}, _capi.BAD_ALIGNMENT), ({"a": P + 8}, _capi.BAD_ALIGNMENT), ({"b": P + 1}, _capi.BAD_ALIGNMENT), ({"output": P + 1}, _capi.BAD_ALIGNMENT),
    ({"rows": P + 2}, _capi.BAD_ALIGNMENT), ({"offsets": P + 1}, _capi.BAD_ALIGNMENT), ({"scale_a": P + 2}, _capi.BAD_ALIGNMENT), ({"scale_a_stride": 2}, _capi.BAD_SHAPE),
    ({"scale_b_stride": 4}, _capi.BAD_SHAPE), ({"rows": None, "count": 6}, _capi.BAD_SHAPE), ({"a_rows": 1 << 26}, _capi.BAD_SHAPE),
    ({"type": _capi.INT8, "k": 131072, "b_stride": 131072}, _capi.BAD_SHAPE), ({"count": 1 << 30, "n": 1 << 21}, _capi.BAD_SHAPE), ({"count": 0, "a_rows": 0}, _capi.SUCCESS),
])
def test_grouped_gemm_refuses_on_the_host(changes, status):
    assert _grouped(**changes) == status


def _int8(**changes):
    args = dict(A=P, B=P, D=P, base=None, base_stride=0, sa=P, sa_stride=1, sb=P, sb_stride=1, m=8, n=32, k=64, b_stride=64, dtype=_capi.BF16, workspace=None,
                bytes=0)
    args.update(changes)
    return LIB.hfrk_int8_gemm(args["A"], args["B"], args["D"], args["base"], args["base_stride"], args["sa"], args["sa_stride"], args["sb"], args["sb_stride"], args["m"],
                              args["n"], args["k"], args["b_stride"], args["dtype"], args["workspace"], args["bytes"], None)


@pytest.mark.parametrize("changes,status", [
    ({"A": None}, _capi.BAD_SHAPE), ({"B": None}, _capi.BAD_SHAPE), ({"D": None}, _capi.BAD_SHAPE), ({"sa": None}, _capi.BAD_SHAPE), ({"m": -1}, _capi.BAD_SHAPE),
    ({"n": 0}, _capi.BAD_SHAPE), ({"k": 40, "b_stride": 48}, _capi.K_NOT_DIVISIBLE_BY_WARPTILE_K), ({"k": 131072, "b_stride": 131072}, _capi.BAD_SHAPE),
    ({"b_stride": 32}, _capi.BAD_SHAPE), ({"b_stride": 65}, _capi.BAD_ALIGNMENT), ({"base": P, "base_stride": 31}, _capi.BAD_SHAPE), ({"base": P + 1}, _capi.BAD_ALIGNMENT),
    ({"dtype": _capi.INT8}, _capi.BAD_DTYPE), ({"sa_stride": -1}, _capi.BAD_SHAPE), ({"m": 0}, _capi.SUCCESS), ({"m": 2 ** 31 - 1, "n": 1 << 21}, _capi.BAD_SHAPE),
])
def test_int8_gemm_refuses_on_the_host(changes, status):
    assert _int8(**changes) == status


def test_int8_gemm_workspace():
    """Few tiles and a long k share it between workgroups; many tiles, few rows and a short k do not."""
    assert LIB.hfrk_int8_gemm_workspace_bytes(128, 4096, 14336) > 0 and LIB.hfrk_int8_gemm_workspace_bytes(64, 4096, 14336) > 0
    for m, n, k in ((1, 4096, 14336), (16, 4096, 14336), (4096, 28672, 4096), (512, 8192, 256), (0, 64, 64), (-1, 64, 64), (100, 0, 64), (1 << 30, 64, 64)):
        assert LIB.hfrk_int8_gemm_workspace_bytes(m, n, k) == 0, (m, n, k)


def _route(**changes):
    args = dict(logits=P, logits_stride=16, bias=None, mask=None, weights=P, experts=P, places=P, rows=P, offsets=P, tokens=4, num_experts=16, top=2, dtype=_capi.FP32,
                sigmoid=0, renormalize=1, factor=1.0)
    args.update(changes)
    memory = args.pop("workspace", None), args.pop("bytes", 0)
    return LIB.hfrk_route_experts(ctypes.byref(_capi.RouteArgs(**args)), *memory, None)


@pytest.mark.parametrize("changes,status", [
    ({"logits": None}, _capi.BAD_SHAPE), ({"weights": None}, _capi.BAD_SHAPE), ({"offsets": None}, _capi.BAD_SHAPE), ({"top": 0}, _capi.BAD_SHAPE), ({"top": 17}, _capi.BAD_SHAPE),
    ({"top": 33, "num_experts": 64}, _capi.BAD_SHAPE), ({"num_experts": 0}, _capi.BAD_SHAPE), ({"num_experts": 513}, _capi.BAD_SHAPE), ({"tokens": -1}, _capi.BAD_SHAPE),
    ({"tokens": (1 << 24) + 1}, _capi.BAD_SHAPE), ({"tokens": 1 << 24, "num_experts": 64, "top": 17}, _capi.BAD_SHAPE), ({"dtype": _capi.INT8}, _capi.BAD_DTYPE),
    ({"logits": P + 2}, _capi.BAD_ALIGNMENT), ({"rows": P + 1}, _capi.BAD_ALIGNMENT), ({"bias": P + 2}, _capi.BAD_ALIGNMENT), ({"logits_stride": -1}, _capi.BAD_SHAPE),
    ({"tokens": 1000}, _capi.EXCEEDS_SCRATCH), ({"tokens": 1000, "workspace": P, "bytes": 127}, _capi.EXCEEDS_SCRATCH),
    ({"tokens": 1000, "workspace": P + 2, "bytes": 4096}, _capi.BAD_ALIGNMENT), ({"bytes": 64}, _capi.EXCEEDS_SCRATCH),
])
def test_route_experts_refuses_on_the_host(changes, status):
    assert _route(**changes) == status


def test_route_experts_workspace():
    sizes = [LIB.hfrk_route_experts_workspace_bytes(*x) for x in ((64, 128, 8), (65, 128, 8), (1000, 16, 2), (1 << 24, 512, 16), (16000, 256, 8), (0, 16, 2), (5, 600, 2))]
    assert sizes == [0, 128 * 4, 2 * 16 * 4, 128 * 512 * 4, 125 * 256 * 4, 0, 0]


def test_combine_and_quantise_refuse_on_the_host():
    def combine(y=P, weights=P, places=P, base=None, output=P, tokens=4, top=2, cols=16, y_rows=8, dtype=_capi.BF16):
        return LIB.hfrk_combine_experts(y, weights, places, base, output, tokens, top, cols, y_rows, dtype, None)

    assert combine(tokens=0) == _capi.SUCCESS
    for changes in ({"y": None}, {"weights": None}, {"places": None}, {"output": None}, {"tokens": -1}, {"tokens": 1 << 24}, {"top": 0}, {"top": 33}, {"cols": 0}, {"cols": (1 << 21) + 1},
                    {"y_rows": -1}):
        assert combine(**changes) == _capi.BAD_SHAPE, changes
    assert combine(dtype=_capi.FP32) == _capi.BAD_DTYPE and combine(y=P + 1) == _capi.BAD_ALIGNMENT and combine(places=P + 2) == _capi.BAD_ALIGNMENT
    assert LIB.hfrk_quantize_int8(P, None, P, None, 2, 16, _capi.BF16, None) == _capi.BAD_SHAPE
    assert LIB.hfrk_quantize_int8(P, None, P, P, 2, 12, _capi.BF16, None) == _capi.BAD_SHAPE
    assert LIB.hfrk_quantize_int8(P, None, P, P, 2, 16, _capi.FP32, None) == _capi.BAD_DTYPE
    assert LIB.hfrk_quantize_int8(P + 2, None, P, P, 2, 16, _capi.BF16, None) == _capi.BAD_ALIGNMENT
    assert LIB.hfrk_quantize_int8(None, None, None, None, 0, 16, _capi.BF16, None) == _capi.SUCCESS
    assert LIB.hfrk_swiglu_dynamic_int8(P, P, None, 2, 16, _capi.BF16, None) == _capi.BAD_SHAPE
    assert LIB.hfrk_swiglu_dynamic_int8(P, P, P, 2, 32776, _capi.BF16, None) == _capi.BAD_SHAPE


def test_wrappers_refuse_tensors_of_the_host():
    w = torch.zeros((2, 32, 64), dtype=INT8)
    with pytest.raises(AssertionError, match="cuda"):
        hf_rocm_kernels.grouped_gemm(torch.zeros((4, 64), dtype=INT8), w.transpose(1, 2), torch.ones(4), None, torch.tensor([0, 2, 4], dtype=torch.int32))
    with pytest.raises(AssertionError, match="cuda"):
        hf_rocm_kernels.int8_gemm(torch.zeros((4, 64), dtype=INT8), w[0].t(), torch.ones(4))
    with pytest.raises(AssertionError, match="cuda"):
        hf_rocm_kernels.route_experts(torch.zeros((4, 8)), 2)
    with pytest.raises(AssertionError, match="scoring"):
        hf_rocm_kernels.route_experts(torch.zeros((4, 8)), 2, scoring="top")
    with pytest.raises(AssertionError, match="cuda"):
        hf_rocm_kernels.combine_experts(torch.zeros((4, 8)).half(), torch.zeros((2, 2)), torch.zeros((2, 2), dtype=torch.int32))
    with pytest.raises(AssertionError):
        hf_rocm_kernels.quantize_int8(torch.zeros((4, 8)).half())
    with pytest.raises(AssertionError, match="next_buffer"):
        hf_rocm_kernels.swiglu_dynamic(torch.zeros((4, 32)).half(), torch.zeros((4, 8)).half(), dtype=INT8)


@pytest.mark.parametrize("codes", [FP8, INT8])
def test_wrappers_under_fake_tensors(codes):
    with FakeTensorMode():
        x = torch.empty((6, 256), dtype=torch.bfloat16, device="cuda")
        q, s = hf_rocm_kernels.quantize_int8(x)
        assert q.dtype == INT8 and s.shape == (6,)
        w, ws = torch.empty((96, 256), dtype=INT8, device="cuda"), torch.empty(96, device="cuda")
        assert hf_rocm_kernels.int8_gemm(q, w.t(), s, ws, out_dtype=torch.float16).dtype == torch.float16
        assert apply_int8_linear(x.view(2, 3, 256), w, ws).shape == (2, 3, 96)
        act, scales = hf_rocm_kernels.swiglu_dynamic(x, dtype=INT8)
        assert act.shape == (6, 128) and act.dtype == INT8 and scales.shape == (6,)
        route = hf_rocm_kernels.route_experts(torch.empty((6, 16), device="cuda"), 4)
        assert route.rows.shape == (24,) and route.offsets.shape == (17,) and route.places.shape == (6, 4)
        gate_up, down = torch.empty((16, 256, 256), dtype=codes, device="cuda"), torch.empty((16, 256, 128), dtype=codes, device="cuda")
        out = expert_mlp_combined_ops(x, torch.empty((6, 16), device="cuda"), 4, gate_up, torch.empty((16, 256), device="cuda"), down, None, residual=x)
        assert out.shape == (6, 256) and out.dtype == torch.bfloat16


def test_int8_quantisation_on_the_host():
    x = torch.tensor([[1.0, -2.0, 0.5, 127.0], [0.0, 0.0, 0.0, 0.0]])
    scale = int8_scale(x, dim=1)
    assert scale[0, 0] == 1.0 and scale[1, 0] == torch.finfo(torch.float32).tiny
    assert int8_quantize(x, scale).tolist() == [[1, -2, 0, 127], [0, 0, 0, 0]]
    layer = Int8Linear.from_float(torch.nn.Linear(32, 8))
    assert layer.weight.dtype == INT8 and layer.weight_scale.shape == (8,) and int(layer.weight.abs().max()) == 127
    assert layer.half().weight_scale.dtype == torch.float32 and "in_features=32" in repr(layer)


def test_plain_forms_make_an_mlp_of_experts():
    """Route, group, multiply, combine, against the sum over a token's experts written out."""
    gen = torch.Generator().manual_seed(0)
    tokens, experts, top, k, n = 9, 5, 2, 32, 8
    logits, a = torch.randn((tokens, experts), generator=gen), torch.randint(-9, 9, (tokens, k), generator=gen, dtype=INT8)
    w, s = torch.randint(-9, 9, (experts, n, k), generator=gen, dtype=INT8), torch.rand(tokens, generator=gen)
    mask = torch.arange(tokens) != 4
    weights, chosen, places, rows, offsets = reference_route_experts(logits, top, mask=mask)
    y = reference_grouped_gemm(a, w.transpose(1, 2), s, None, offsets, rows=rows)
    out = reference_combine_experts(y, weights, places)
    for t in range(tokens):
        best = torch.topk(logits[t].double(), top)
        p = torch.softmax(best.values, 0)
        expected = sum(p[j] * (w[best.indices[j]].double() @ a[t].double()) * s[t].double() for j in range(top)) if bool(mask[t]) else torch.zeros(n).double()
        assert torch.allclose(out[t], expected, rtol=1e-12)
