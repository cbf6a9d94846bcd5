"""The router, the experts' sum, and an MLP of experts made of them, against plain forms in 64 bits."""
import math

import pytest
import torch

from hf_rocm_kernels import combine_experts, grouped_gemm, quantize_fp8, quantize_int8, route_experts, swiglu_dynamic
from hf_rocm_kernels.combined_ops.expert_mlp import expert_mlp_combined_ops
from hf_rocm_kernels.operators.experts import reference_combine_experts, reference_route_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
INT8 = torch.int8


def _check(route, logits, top, experts_exact=True, **options):
    weights, experts, places, rows, offsets = reference_route_experts(logits, top, **{k: (v.cpu() if torch.is_tensor(v) else v) for k, v in options.items()})
    assert torch.equal(route.experts.cpu(), experts)
    assert torch.equal(route.places.cpu(), places) and torch.equal(route.rows.cpu(), rows) and torch.equal(route.offsets.cpu(), offsets)
    got = route.weights.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(weights))
    # fp32: an exponential of an argument rounded at up to 32 (2^-19 relative), sums of up to 512 terms along chains of 8 + 6, divisions
    fine = ~torch.isnan(weights)
    assert ((got - weights).abs()[fine] <= 2.0 ** -18 * weights.abs()[fine] + 1e-37).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (1, 128, 8), (3, 5, 5), (17, 8, 2), (64, 60, 4), (65, 64, 6), (128, 512, 8), (300, 65, 32), (200, 256, 10),
                                                (1000, 130, 1)])
def test_route(dtype, tokens, experts, top):
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    logits = (2 * torch.randn((tokens, experts), generator=gen, device=DEV)).to(dtype)
    for options in ({}, {"scoring": "sigmoid", "renormalize": False, "factor": 2.5}, {"renormalize": False}, {"scoring": "sigmoid"}):
        _check(route_experts(logits, top, **options), logits, top, **options)


def _many(logits, top, scoring, bias, mask=None):
    """A route of many tokens by sorts in 64 bits: (experts, places, rows, offsets)."""
    x = logits.double()
    key = x if bias is None else (torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)) + bias.double()
    key = torch.where((x > -math.inf) & (key > -math.inf), key, -math.inf)
    order = torch.sort(key, dim=1, descending=True, stable=True)
    experts = torch.where(order.values[:, :top] > -math.inf, order.indices[:, :top], -1)
    if mask is not None:
        experts = torch.where(mask[:, None], experts, -1)
    flat = experts.reshape(-1)
    group = torch.where(flat < 0, logits.size(1), flat)
    pairs = torch.sort(group, stable=True).indices
    offsets = torch.searchsorted(group[pairs], torch.arange(logits.size(1) + 1, device=DEV))
    held = torch.arange(flat.numel(), device=DEV) < offsets[-1]
    places = torch.empty_like(flat)
    places[pairs] = torch.where(held, torch.arange(flat.numel(), device=DEV), -1)
    return experts, places.view_as(experts), torch.where(held, pairs // top, -1), offsets


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,experts,top", [(2049, 4, 4), (3000, 60, 6), (2500, 64, 17), (4097, 128, 8), (2050, 129, 32), (5000, 256, 8), (16001, 200, 3), (2100, 384, 10)])
def test_route_of_many_tokens(dtype, tokens, experts, top):
    """bfloat16 logits repeat, so ties are many; a bias leaves choices that 32 bits cannot tell."""
    gen = torch.Generator(device=DEV).manual_seed(tokens + top)
    logits = (2 * torch.randn((tokens, experts + 3), generator=gen, device=DEV)).to(dtype)[:, 1:experts + 1]
    logits[7] = -math.inf
    logits[8, experts // 2:] = -math.inf
    logits[9, 1] = math.nan
    bias = 0.1 * torch.randn(experts, generator=gen, device=DEV)
    bias[experts // 3] = bias[0] * (1 + 2.0 ** -22)  # sums one step of 32 bits apart
    mask = torch.rand(tokens, generator=gen, device=DEV) < 0.9
    for scoring, b, m in (("softmax", None, None), ("softmax", bias, mask), ("sigmoid", bias, None), ("sigmoid", None, mask)):
        clean = torch.where(torch.isnan(logits), -math.inf, logits.float()).to(dtype)  # what is none is not chosen
        route = route_experts(logits, top, bias=b, scoring=scoring, mask=m)
        wanted = _many(clean, top, scoring, b, m)
        if b is not None:  # the NaN in a softmax's sum leaves that row without a choice
            keep = torch.arange(tokens, device=DEV) != 9
            assert torch.equal(route.experts[keep].long(), wanted[0][keep])
        else:
            for got, want in zip((route.experts, route.places, route.rows, route.offsets), wanted):
                assert torch.equal(got.long(), want)
        score = torch.softmax(clean.double(), 1) if scoring == "softmax" else torch.sigmoid(clean.double())
        weights = score.gather(1, wanted[0].clamp(min=0)).masked_fill(wanted[0] < 0, 0.0)
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
        real = torch.ones(tokens, dtype=torch.bool, device=DEV) if m is None else m.clone()
        if bool(real[9]):
            assert torch.isnan(route.weights[9]).all()
        rest = torch.arange(tokens, device=DEV) != 9
        rest[7] = False
        # as in _check, and the choices' sum
        assert ((route.weights.double() - weights).abs()[rest] <= 2.0 ** -17 * weights[rest] + 1e-37).all()
        assert (route.weights[7] == 0).all() and (route.weights[~real] == 0).all()


@pytest.mark.parametrize("tokens", [100, 3000])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_with_a_bias_that_32_bits_cannot_tell(tokens, scoring):
    """Sums that are equal in 32 bits and not in 64, and sums that are equal in both."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    logits = torch.randn((tokens, 96), generator=gen, device=DEV) * 2.0 ** -14
    bias = torch.full((96,), 4.0, device=DEV)
    route = route_experts(logits, 6, bias=bias, scoring=scoring)
    wanted = _many(logits, 6, scoring, bias)
    for got, want in zip((route.experts, route.places, route.rows, route.offsets), wanted):
        assert torch.equal(got.long(), want)
    same = route_experts(torch.zeros_like(logits), 6, bias=bias, scoring=scoring)
    assert (same.experts == torch.arange(6, device=DEV)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,top", [(5, 16, 3), (100, 200, 8), (400, 65, 4)])
def test_route_with_a_bias_and_padding(scoring, tokens, experts, top):
    gen = torch.Generator(device=DEV).manual_seed(top)
    wide = torch.randn((tokens, experts + 7), generator=gen, device=DEV)
    logits = wide[:, 3:3 + experts]  # rows further apart than they are long
    bias = 0.2 * torch.randn(experts, generator=gen, device=DEV)
    mask = torch.rand(tokens, generator=gen, device=DEV) < 0.8
    route = route_experts(logits, top, bias=bias, scoring=scoring, mask=mask, factor=1.5)
    _check(route, logits, top, bias=bias, scoring=scoring, mask=mask, factor=1.5)
    again = route_experts(logits, top, bias=bias, scoring=scoring, mask=mask.to(torch.uint8), factor=1.5)
    assert all(torch.equal(x, y) for x, y in zip(route, again))


@pytest.mark.parametrize("tokens", [4, 300])
def test_route_ties_go_to_the_lowest_index(tokens):
    logits = torch.zeros((tokens, 100), device=DEV, dtype=torch.bfloat16)
    logits[:, 1::2] = -0.0  # both zeros are one
    logits[1::2, 70] = 1.0
    route = route_experts(logits, 3)
    _check(route, logits, 3)
    assert route.experts[0].tolist() == [0, 1, 2] and route.experts[1].tolist() == [70, 0, 1]
    sure = torch.full((tokens, 100), 30.0, device=DEV)  # scores are all 1 in fp32, the logits are not
    sure[:, 9] = 31.0
    assert route_experts(sure, 2, scoring="sigmoid").experts[0].tolist() == [9, 0]


@pytest.mark.parametrize("tokens", [6, 200])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_infinities_and_nan(tokens, scoring):
    gen = torch.Generator(device=DEV).manual_seed(0)
    logits = torch.randn((tokens, 70), generator=gen, device=DEV)
    logits[0] = -math.inf                      # nothing is left
    logits[1, :68] = -math.inf                 # two are left, four are asked for
    logits[2, 5] = math.nan
    logits[3] = math.nan
    logits[4, 1:] = torch.finfo(torch.float32).min
    for bias in (None, torch.zeros(70, device=DEV).index_fill_(0, torch.tensor([69], device=DEV), -math.inf)):
        route = route_experts(logits, 4, bias=bias, scoring=scoring)
        _check(route, logits, 4, bias=bias, scoring=scoring)
        assert route.experts[0].tolist() == [-1] * 4 and (route.weights[0] == 0).all()
        assert torch.isnan(route.weights[2]).all() and 5 not in route.experts[2].tolist()
        if bias is not None:
            assert not (route.experts == 69).any()
    nothing = route_experts(logits[:0], 4)
    assert nothing.offsets.tolist() == [0] * 71 and nothing.rows.numel() == 0
    none = route_experts(logits, 4, mask=torch.zeros(tokens, dtype=torch.bool, device=DEV))
    assert (none.experts == -1).all() and (none.rows == -1).all() and (none.places == -1).all() and (none.weights == 0).all() and (none.offsets == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,top,cols", [(1, 1, 1), (5, 8, 2048), (3, 2, 7), (33, 6, 264), (200, 9, 1000), (64, 32, 4104), (7, 3, 2049)])
def test_combine(dtype, tokens, top, cols):
    gen = torch.Generator(device=DEV).manual_seed(cols)
    y = torch.randn((tokens * top, cols), generator=gen, device=DEV).to(dtype)
    places = torch.randperm(tokens * top, generator=gen, device=DEV).int().reshape(tokens, top)
    places[0, 0] = -1
    places[-1, -1] = tokens * top  # no row
    weights = torch.rand((tokens, top), generator=gen, device=DEV)
    base = torch.randn((tokens, cols), generator=gen, device=DEV).to(dtype)
    for add in (None, base):
        out = combine_experts(y, weights, places, base=add)
        exact = reference_combine_experts(y, weights, places, add)
        magnitude = reference_combine_experts(y.abs(), weights, places, None if add is None else add.abs())
        # one rounding to 16 bits; top products and sums in fp32
        bound = torch.finfo(dtype).eps / 2 * (exact.abs() + 1e-4 * magnitude) + (top + 2) * 2.0 ** -24 * magnitude + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert ((out.double() - exact).abs() <= bound).all()
        into = torch.empty_like(out)
        assert combine_experts(y, weights, places, base=add, output=into) is into and torch.equal(into, out)
    shared = base.clone()
    assert torch.equal(combine_experts(y, weights, places, base=shared, output=shared), out)


def test_combine_keeps_nan_and_ignores_rows_that_are_not_named():
    y = torch.full((4, 16), math.nan, device=DEV, dtype=torch.bfloat16)
    y[2] = 2.0
    weights, places = torch.tensor([[0.5, 0.0], [0.0, 0.0], [math.nan, 0.0]], device=DEV), torch.tensor([[2, -1], [-1, -1], [-1, -1]], device=DEV, dtype=torch.int32)
    out = combine_experts(y, weights, places)
    assert (out[0] == 1.0).all() and (out[1] == 0.0).all() and torch.isnan(out[2]).all()
    assert combine_experts(y[:0], weights[:2], places[:2]).abs().max() == 0
    assert combine_experts(y, weights[:0], places[:0]).shape == (0, 16)


def test_refusals():
    logits = torch.zeros((4, 8), device=DEV)
    for bad in (lambda: route_experts(logits, 0), lambda: route_experts(logits, 9), lambda: route_experts(logits.double(), 2), lambda: route_experts(logits[0], 1),
                lambda: route_experts(logits, 2, scoring="tanh"), lambda: route_experts(logits, 2, bias=torch.zeros(7, device=DEV)),
                lambda: route_experts(logits, 2, bias=torch.zeros(8, device=DEV).half()), lambda: route_experts(logits, 2, mask=torch.ones(3, device=DEV).bool()),
                lambda: route_experts(logits.t().contiguous().t(), 2), lambda: route_experts(torch.zeros((2, 513), device=DEV), 2),
                lambda: route_experts(torch.zeros((2, 100), device=DEV), 33), lambda: route_experts(logits.cpu(), 2)):
        with pytest.raises((AssertionError, RuntimeError)):
            bad()
    y, weights, places = torch.zeros((8, 16), device=DEV).half(), torch.zeros((4, 2), device=DEV), torch.zeros((4, 2), device=DEV, dtype=torch.int32)
    for bad in (lambda: combine_experts(y.float(), weights, places), lambda: combine_experts(y, weights.half(), places), lambda: combine_experts(y, weights, places.long()),
                lambda: combine_experts(y, weights[:3], places), lambda: combine_experts(y, weights, places, base=y[:3]), lambda: combine_experts(y[:, ::2], weights, places),
                lambda: combine_experts(y, weights, places, base=torch.zeros((4, 16), device=DEV)), lambda: combine_experts(y, weights.cpu(), places),
                lambda: combine_experts(y, torch.zeros((4, 33), device=DEV), torch.zeros((4, 33), device=DEV, dtype=torch.int32)),
                lambda: combine_experts(y, weights, places, output=y[:4])):
        with pytest.raises((AssertionError, RuntimeError)):
            bad()


def _plain_mlp(x, logits, top, gate_up, gate_up_scale, down, down_scale, residual, mask):
    """In 64 bits but for the roundings that the operators make: codes of the inputs and of the activations, 16-bit projections."""
    int8 = gate_up.dtype == INT8
    most = 127.0 if int8 else 448.0
    inter = down.size(2)

    def codes(v, code_dtype):
        scale = (v.abs().amax(1, keepdim=True) / most).clamp(min=1e-30)
        q = v / scale
        return (q.round() if int8 else q.float().to(FP8).double()) * scale

    weights, experts, _, _, _ = reference_route_experts(logits, top, mask=mask)
    x = codes(x.double(), gate_up.dtype)
    out = torch.zeros_like(x) if residual is None else residual.double().clone()
    for t in range(x.size(0)):
        for j in range(top):
            e = int(experts[t, j])
            if e < 0:
                continue
            g = (gate_up[e].float().double() * gate_up_scale[e].double()[:, None]) @ x[t]
            gate, up = g[:inter], g[inter:]
            h = codes((gate * torch.sigmoid(gate) * up)[None], gate_up.dtype)[0]
            out[t] += float(weights[t, j]) * ((down[e].float().double() * down_scale[e].double()[:, None]) @ h)
    return out


@pytest.mark.parametrize("codes", [FP8, INT8])
@pytest.mark.parametrize("tokens,experts,top,hidden,inter", [(1, 8, 2, 256, 128), (6, 16, 4, 128, 96), (150, 5, 2, 192, 160)])
def test_mlp_of_experts(codes, tokens, experts, top, hidden, inter):
    """The set as it is used, eagerly, then captured and replayed with other contents."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)

    def weight(n, k):
        w = torch.randn((experts, n, k), generator=gen, device=DEV) * k ** -0.5
        scale = w.abs().amax(2) / (127.0 if codes == INT8 else 448.0)
        w = w / scale[..., None]
        return (w.round().to(INT8) if codes == INT8 else w.to(FP8)), scale

    (gate_up, gate_up_scale), (down, down_scale) = weight(2 * inter, hidden), weight(hidden, inter)
    x = torch.randn((tokens, hidden), generator=gen, device=DEV).bfloat16()
    logits = torch.randn((tokens, experts), generator=gen, device=DEV)
    residual = torch.randn((tokens, hidden), generator=gen, device=DEV).bfloat16()
    mask = torch.ones(tokens, dtype=torch.bool, device=DEV)
    mask[tokens // 2 + 1:tokens // 2 + 2] = False

    def call():
        return expert_mlp_combined_ops(x, logits, top, gate_up, gate_up_scale, down, down_scale, residual=residual, mask=mask)

    def check(out):
        exact = _plain_mlp(x, logits, top, gate_up, gate_up_scale, down, down_scale, residual, mask)
        mlp = (exact - residual.double()).abs().max()
        # the projections and the sum are rounded to 16 bits (2^-8 each) in front of sums over hidden values of either sign; the activations' codes can
        # move to a neighbour by that (int8: a step is 1/127 of the largest; fp8: 2^-3 of the value), one in some
        step = 2.0 ** -8 * 4 + (1 / 127 if codes == INT8 else 2.0 ** -4)
        assert ((out.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + step * mlp).all()
        assert torch.equal(out[~mask], residual[~mask])

    eager = call()
    check(eager)
    q, s = quantize_int8(x) if codes == INT8 else quantize_fp8(x)  # the same operators one by one
    route = route_experts(logits, top, mask=mask)
    h, hs = swiglu_dynamic(grouped_gemm(q, gate_up.transpose(1, 2), s, gate_up_scale, route.offsets, rows=route.rows), dtype=codes)
    y = grouped_gemm(h, down.transpose(1, 2), hs, down_scale, route.offsets)
    assert torch.equal(combine_experts(y, route.weights, route.places, base=residual), eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        x.copy_(torch.randn((tokens, hidden), generator=gen, device=DEV))
        logits.copy_(torch.randn((tokens, experts), generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
    check(out)


@pytest.mark.parametrize("codes", [FP8, INT8])
def test_traced_mlp_of_experts_equals_the_eager_one(codes):
    gen = torch.Generator(device=DEV).manual_seed(3)
    experts, hidden, inter = 6, 128, 64

    def weight(n, k):
        w = torch.randint(-120, 121, (experts, n, k), generator=gen, device=DEV, dtype=torch.int8)
        return (w if codes == INT8 else (w.float() / 64).to(FP8)), torch.rand((experts, n), generator=gen, device=DEV) / 64

    (gate_up, gate_up_scale), (down, down_scale) = weight(2 * inter, hidden), weight(hidden, inter)
    bias = torch.rand(experts, generator=gen, device=DEV)

    def block(x, logits):
        return expert_mlp_combined_ops(x, logits, 3, gate_up, gate_up_scale, down, down_scale, residual=x, bias=bias, scoring="sigmoid")

    traced = torch.compile(block, backend="aot_eager", fullgraph=True)
    for tokens in (1, 9, 9, 80):
        x, logits = torch.randn((tokens, hidden), generator=gen, device=DEV).bfloat16(), torch.randn((tokens, experts), generator=gen, device=DEV)
        assert torch.equal(traced(x, logits), block(x, logits)), tokens


def test_two_blocks_at_once_do_not_meet():
    """Two captured blocks replayed side by side, each with its own workspaces, and eager calls between them."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    experts, hidden, inter, tokens, top = 64, 256, 128, 300, 4
    gate_up = torch.randint(-127, 128, (experts, 2 * inter, hidden), generator=gen, device=DEV, dtype=torch.int8)
    down = torch.randint(-127, 128, (experts, hidden, inter), generator=gen, device=DEV, dtype=torch.int8)
    s1, s2 = torch.rand((experts, 2 * inter), generator=gen, device=DEV) / 512, torch.rand((experts, hidden), generator=gen, device=DEV) / 512
    x = [torch.randn((tokens, hidden), generator=gen, device=DEV).half() for _ in range(2)]
    logits = [torch.randn((tokens, experts), generator=gen, device=DEV) for _ in range(2)]

    def call(i):
        return expert_mlp_combined_ops(x[i], logits[i], top, gate_up, s1, down, s2)

    call(0)
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for _ in range(5):
        for i in range(2):
            x[i].copy_(torch.randn((tokens, hidden), generator=gen, device=DEV))
            logits[i].copy_(torch.randn((tokens, experts), generator=gen, device=DEV))
        want = [call(i) for i in range(2)]
        torch.cuda.synchronize()
        eager = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
                eager.append(call(1 - i))
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) and torch.equal(eager[i], want[1 - i]) for i in range(2))


def test_route_and_combine_of_the_most_tokens():
    gen = torch.Generator(device=DEV).manual_seed(5)
    tokens = 1 << 24
    logits = torch.randn((tokens, 3), generator=gen, device=DEV)
    route = route_experts(logits, 1)
    best = logits.argmax(1)
    assert torch.equal(route.experts[:, 0].long(), best) and (route.weights == 1.0).all()
    order = torch.sort(best, stable=True).indices
    assert torch.equal(route.rows.long(), order) and torch.equal(route.places[order, 0].long(), torch.arange(tokens, device=DEV))
    assert route.offsets.tolist() == [0, *torch.bincount(best, minlength=3).cumsum(0).tolist()]
    tokens -= 1
    y = torch.randn((1000, 8), generator=gen, device=DEV).bfloat16()
    places = torch.randint(-1, 1000, (tokens, 1), generator=gen, device=DEV, dtype=torch.int32)
    out = combine_experts(y, torch.full((tokens, 1), 0.5, device=DEV), places)
    assert torch.equal(out, torch.where(places < 0, 0.0, y[places[:, 0].clamp(min=0).long()] * 0.5).bfloat16())
