"""Products grouped by expert, products of int8 codes and their linear layers, against plain forms in 64 bits.

Tolerances.  A result is rounded once to 16 bits: half a step, eps / 2 relative.  In front of that the sum S is converted (int8: exact, then one
rounding to fp32, 2^-24), multiplied by the product of the two scales (two roundings) and added to the addend (one): 4 * 2^-24 of |S sa sb| + |base|.  fp8 sums
are made by the matrix cores.  They align a run of eight products to the largest of them and cut what is below 2^-13 of its power of two (seen on the card:
x + y - x is y down to y = 2^-13 x and 0 below, for x and y in one run of eight, and y down to 2^-23 x in different ones), so each run loses less than 7 * 2^-13
of its largest product; runs are then added in fp32: at most k * 2^-23 of the sum of magnitudes (2^-23, not 2^-24, where they cut instead of rounding)."""
import pytest
import torch

import hf_rocm_kernels
from hf_rocm_kernels import _capi
from hf_rocm_kernels import grouped_gemm, int8_gemm, quantize_int8, swiglu_dynamic
from hf_rocm_kernels.layers import Int8Linear, apply_int8_linear, convert_linear_layers
from hf_rocm_kernels.operators.grouped_gemm import reference_grouped_gemm
from hf_rocm_kernels.operators.int8_gemm import reference_int8_gemm
from hf_rocm_kernels.operators.quantize import reference_quantize_int8

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
INT8 = torch.int8


def _codes(gen, shape, dtype):
    if dtype == INT8:
        return torch.randint(-127, 128, shape, generator=gen, device=DEV, dtype=torch.int8)
    return torch.randn(shape, generator=gen, device=DEV).mul_(60).clamp_(-448, 448).to(FP8)


def _scales(gen, *shape):
    return 0.001 + 0.01 * torch.rand(shape, generator=gen, device=DEV)


def _close(out, exact, magnitude, k, codes, base=None, cut=0.0):
    """magnitude: the sum of magnitudes with the scales applied; cut: what the runs of eight fp8 products lose (_cut)."""
    eps = torch.finfo(out.dtype).eps / 2
    tiny = torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    slack = cut + (k * 2.0 ** -23 if codes == FP8 else 0.0) * magnitude + 4 * 2.0 ** -24 * (magnitude + (0 if base is None else base.double().abs()))
    bound = eps * (exact.abs() + slack) + slack + tiny
    wrong = (out.double() - exact).abs() > bound
    assert not wrong.any(), (int(wrong.sum()), (out.double() - exact).abs().max(), wrong.nonzero()[:4])


def _magnitude(a, w, sa, sb):
    """sum_k |a| |w| with scales; a (m, k), w (n, k)."""
    out = (a.float().abs().double() @ w.float().abs().double().t()) * sa.double().reshape(-1, 1)
    return out if sb is None else out * sb.double().reshape(1, -1)


def _cut(a, w, sa, sb):
    """7 * 2^-13 of the largest product of every eight, summed; a (m, k), w (n, k) in fp8 (int8: nothing is cut)."""
    if a.dtype != FP8:
        return 0.0
    m, n, k = a.size(0), w.size(0), a.size(1)
    out = torch.empty((m, n), dtype=torch.float64, device=a.device)
    step = max(1, (1 << 26) // (n * k))
    for i in range(0, m, step):
        products = a[i:i + step].float().abs()[:, None] * w.float().abs()[None]
        out[i:i + step] = products.view(-1, n, k // 8, 8).amax(-1).double().sum(-1)
    out = out * (7 * 2.0 ** -13) * sa.double().reshape(-1, 1)
    return out if sb is None else out * sb.double().reshape(1, -1)


def _grouped(sizes, k, n, codes, dtype, gather, seed=0, front=0, behind=0, experts_of=None, scale_b="channel"):
    """Run a call and compare every group; returns nothing.  front, behind: rows of the result that belong to no group."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    experts, count = len(sizes), sum(sizes) + front + behind
    offsets = torch.tensor([front] + [front + sum(sizes[:e + 1]) for e in range(experts)], dtype=torch.int32, device=DEV)
    tokens = max(1, count // 3) if gather else count
    a, w = _codes(gen, (tokens, k), codes), _codes(gen, (experts, n, k), codes)
    sa = _scales(gen, tokens)
    sb = {"channel": lambda: _scales(gen, experts, n), "expert": lambda: _scales(gen, experts), "none": lambda: None}[scale_b]()
    rows = torch.randint(0, tokens, (count,), generator=gen, device=DEV, dtype=torch.int32) if gather else None
    output = torch.full((count, n), 7.0, dtype=dtype, device=DEV)
    back = grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows, output=output)
    assert back is output
    first = front
    for e, size in enumerate(sizes):
        here = slice(first, first + size)
        index = torch.arange(first, first + size, device=DEV) if rows is None else rows[here].long()
        ae = a.view(torch.uint8)[index].view(a.dtype)
        s = None if sb is None else sb[e]
        if size:
            exact = reference_int8_gemm(ae.float(), w[e].float().t(), sa[index], s)
            _close(output[here], exact, _magnitude(ae, w[e], sa[index], s), k, codes, cut=_cut(ae, w[e], sa[index], s))
        first += size
    assert (output[:front] == 7.0).all() and (output[first:] == 7.0).all()
    again = grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows, out_dtype=dtype)
    assert torch.equal(again[front:first], output[front:first])  # equal calls, equal bits


@pytest.mark.parametrize("codes", [FP8, INT8])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("sizes,k,n", [
    ([1], 16, 1), ([1, 0, 2], 48, 7), ([0, 0, 0], 64, 16), ([3, 1, 16, 17, 0, 33], 128, 40), ([5, 64, 65, 1], 272, 72),
    ([2] * 70, 144, 24), ([0] * 63 + [9, 1], 256, 32), ([1, 300, 0, 128, 129, 31], 1040, 136), ([0, 511, 2], 512, 264), ([1] * 8, 2048, 1536),
    ([257, 256, 255], 640, 520), ([16] * 512, 32, 8),
])
def test_grouped(codes, gather, sizes, k, n):
    _grouped(sizes, k, n, codes, torch.bfloat16, gather, seed=len(sizes) + k)


@pytest.mark.parametrize("codes", [FP8, INT8])
@pytest.mark.parametrize("sizes", [[40, 0, 3], [200, 77, 0, 500], [900, 700, 800]])
def test_grouped_rows_of_no_group_are_left_alone(codes, sizes):
    _grouped(sizes, 256, 96, codes, torch.float16, False, front=5, behind=11)
    _grouped(sizes, 256, 101, codes, torch.float16, True, front=3, behind=300)


@pytest.mark.parametrize("scale_b", ["expert", "none"])
@pytest.mark.parametrize("size", [6, 150])
def test_grouped_scales_of_other_forms(scale_b, size):
    _grouped([size, 4, 0, size], 192, 64, INT8, torch.float16, False, scale_b=scale_b)
    _grouped([size, 4, 0, size], 192, 64, FP8, torch.bfloat16, True, scale_b=scale_b)


@pytest.mark.parametrize("size", [3, 90, 400])
def test_grouped_weights_with_strides_and_one_scale(size):
    gen = torch.Generator(device=DEV).manual_seed(3)
    k, n = 160, 56
    whole = _codes(gen, (3, n + 8, k + 32), INT8)
    w = whole[:, 8:, :k]  # rows and experts further apart than they are long
    a, one = _codes(gen, (2 * size, k), INT8), torch.tensor([0.01], device=DEV)
    sb = _scales(gen, 3, n + 16)[:, :n]
    offsets = torch.tensor([0, size, size, 2 * size], dtype=torch.int32, device=DEV)
    out = grouped_gemm(a, w.transpose(1, 2), one, sb, offsets, out_dtype=torch.float16)
    exact = reference_grouped_gemm(a, w.transpose(1, 2), one, sb, offsets)
    magnitude = torch.cat([_magnitude(a[:size], w[0], one, sb[0]), _magnitude(a[size:], w[2], one, sb[2])])
    _close(out, exact, magnitude, k, INT8)


@pytest.mark.parametrize("size", [4, 130])
def test_grouped_row_numbers_that_are_no_rows_give_zeros(size):
    gen = torch.Generator(device=DEV).manual_seed(4)
    a, w = _codes(gen, (9, 128), FP8), _codes(gen, (2, 32, 128), FP8)
    rows = torch.randint(0, 9, (2 * size,), generator=gen, device=DEV, dtype=torch.int32)
    rows[1], rows[size], rows[-1] = -1, 9, 2 ** 31 - 1
    offsets = torch.tensor([0, size, 2 * size], dtype=torch.int32, device=DEV)
    sa, sb = _scales(gen, 9), _scales(gen, 2, 32)
    out = grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows)
    assert (out[[1, size, 2 * size - 1]] == 0).all()
    exact = reference_grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows)
    index = rows.long().clamp(0, 8)
    for e, here in enumerate((slice(0, size), slice(size, 2 * size))):
        good = ((rows[here] >= 0) & (rows[here] < 9)).nonzero().flatten()
        ae, se = a.view(torch.uint8)[index[here][good]].view(FP8), sa[index[here][good]]
        _close(out[here][good], exact[here][good], _magnitude(ae, w[e], se, sb[e]), 128, FP8, cut=_cut(ae, w[e], se, sb[e]))


@pytest.mark.parametrize("n", [32, 31])
@pytest.mark.parametrize("size", [4, 130])
def test_grouped_scales_of_other_rows_do_not_reach_rows_that_are_none(size, n):
    """The first row's scale is infinite: rows that pick no row of `a` are zero, those that pick another one are that row's."""
    gen = torch.Generator(device=DEV).manual_seed(14)
    a, w = _codes(gen, (9, 128), INT8), _codes(gen, (2, n, 128), INT8)
    rows = torch.randint(1, 9, (2 * size,), generator=gen, device=DEV, dtype=torch.int32)
    none = [0, 2, size, 2 * size - 1]
    rows[none] = torch.tensor([-1, 9, -2 ** 31, 1 << 29], dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, size, 2 * size], dtype=torch.int32, device=DEV)
    sa = _scales(gen, 9)
    sa[0] = float("inf")
    out = grouped_gemm(a, w.transpose(1, 2), sa, None, offsets, rows=rows)
    assert (out[none] == 0).all() and out.isfinite().all()
    for e, here in enumerate((slice(0, size), slice(size, 2 * size))):
        good = ((rows[here] > 0) & (rows[here] < 9)).nonzero().flatten()
        picked = rows[here][good].long()
        exact = reference_int8_gemm(a[picked], w[e].t(), sa[picked])
        _close(out[here][good], exact, _magnitude(a[picked], w[e], sa[picked], None), 128, INT8)


@pytest.mark.parametrize("offsets", [[0, 50, 20, 60], [-5, 10, 10, 999], [60, 0, 0, 60], [2 ** 31 - 1, -2 ** 31, 30, 60]])
def test_grouped_offsets_that_are_none_stay_inside(offsets):
    """Broken offsets give no answer, and reach no memory that is not the call's: what lies around the result stays as it was."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    a, w = _codes(gen, (60, 64), INT8), _codes(gen, (3, 16, 64), INT8)
    around = torch.full((80, 16), 7.0, dtype=torch.bfloat16, device=DEV)
    grouped_gemm(a, w.transpose(1, 2), _scales(gen, 60), None, torch.tensor(offsets, dtype=torch.int32, device=DEV), output=around[10:70])
    assert (around[:10] == 7.0).all() and (around[70:] == 7.0).all()


@pytest.mark.parametrize("m", [0, 1, 2, 5, 16, 17, 32, 33, 48, 64, 65, 100, 129, 256, 300, 1000])
@pytest.mark.parametrize("n,k,base", [(8, 16, None), (1, 128, "row"), (100, 272, "full"), (1000, 1024, "row"), (520, 4112, None), (257, 640, "full")])
def test_int8_gemm(m, n, k, base):
    gen = torch.Generator(device=DEV).manual_seed(m + n)
    dtype = torch.bfloat16 if (m + n) % 2 else torch.float16
    a, w = _codes(gen, (m, k), INT8), _codes(gen, (n, k), INT8)
    sa, sb = _scales(gen, m) if m != 1 else _scales(gen, 1), _scales(gen, n)
    add = {None: None, "row": torch.randn(n, generator=gen, device=DEV).to(dtype), "full": torch.randn((m, n), generator=gen, device=DEV).to(dtype)}[base]
    out = int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype)
    exact = reference_int8_gemm(a, w.t(), sa, sb, add)
    _close(out, exact, _magnitude(a, w, sa, sb), k, INT8, add)
    into = torch.empty((m, n), dtype=dtype, device=DEV)
    assert int8_gemm(a, w.t(), sa, sb, base=add, output=into) is into and torch.equal(into, out)


@pytest.mark.parametrize("m", [1, 3, 4, 5, 8, 9, 13, 16, 17, 20, 24, 25, 32])
@pytest.mark.parametrize("n,k,base", [(1024, 512, None), (1030, 768, "row"), (1027, 1280, "full"), (2304, 4096, "full"), (6148, 512, "row"), (5120, 8192, None), (9218, 1024, "row")])
def test_int8_gemm_on_bands_of_rows(m, n, k, base):
    gen = torch.Generator(device=DEV).manual_seed(m + n)
    dtype = torch.bfloat16 if (m + n) % 2 else torch.float16
    a, wide = _codes(gen, (m, k), INT8), _codes(gen, (n, k + 32), INT8)
    w = wide[:, :k] if m % 2 else wide[:, :k].contiguous()  # rows further apart than they are long
    sa, sb = _scales(gen, m) if m != 4 else _scales(gen, 1), _scales(gen, n) if m != 8 else None
    add = {None: None, "row": torch.randn(n, generator=gen, device=DEV).to(dtype), "full": torch.randn((m, n), generator=gen, device=DEV).to(dtype)}[base]
    out = int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype)
    exact = reference_int8_gemm(a, w.t(), sa, sb, add)
    _close(out, exact, _magnitude(a, w, sa, sb), k, INT8, add)
    assert torch.equal(int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype), out)
    if base == "full":
        assert int8_gemm(a, w.t(), sa, sb, base=add, output=add) is add and torch.equal(add, out)


@pytest.mark.parametrize("m", [17, 24, 32, 33, 47, 48, 49, 64])
@pytest.mark.parametrize("n,k,base", [(8, 2048, None), (1000, 4096, "row"), (1027, 2048, "full"), (4104, 4096, "full"), (6144, 4096, None), (9218, 2048, "row")])
def test_int8_gemm_with_rows_in_registers(m, n, k, base):
    gen = torch.Generator(device=DEV).manual_seed(m + n)
    dtype = torch.bfloat16 if (m + n) % 2 else torch.float16
    a, wide = _codes(gen, (m, k), INT8), _codes(gen, (n, k + 48), INT8)
    w = wide[:, :k] if m % 2 else wide[:, :k].contiguous()
    a[0], w[0] = -128, -128  # a sum of 2^14 k: not a float's
    a[0, 0] = 127
    sa, sb = _scales(gen, m) if m != 48 else _scales(gen, 1), _scales(gen, n) if m != 32 else None
    sa = sa * (1.0 if m != 32 else 2.0 ** -10)  # (within float16)
    add = {None: None, "row": torch.randn(n, generator=gen, device=DEV).to(dtype), "full": torch.randn((m, n), generator=gen, device=DEV).to(dtype)}[base]
    out = int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype)
    exact = reference_int8_gemm(a, w.t(), sa, sb, add)
    _close(out, exact, _magnitude(a, w, sa, sb), k, INT8, add)
    assert torch.equal(int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype), out)
    if base == "full":
        assert int8_gemm(a, w.t(), sa, sb, base=add, output=add) is add and torch.equal(add, out)


@pytest.mark.parametrize("m", [3, 16, 32])
def test_int8_gemm_on_bands_largest_sums(m):
    """Sums above 2^24 that several waves make together stay exact up to the rounding of the result: 2^14 * 130816 and one less, over k in eight parts."""
    k, n = 130816, 1024
    a = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    w[2, ::2] = 127
    w[3, -256:] = 1
    one = torch.ones(1, device=DEV) * 2.0 ** -20
    out = int8_gemm(a, w.t(), one, out_dtype=torch.float16)
    exact = reference_int8_gemm(a[:1], w[:8].t(), one)
    bound = exact.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25  # the sum made a float, times one scale, rounded to fp16
    assert ((out[:, :8].double() - exact).abs() <= bound).all()
    assert (out == out[:1]).all() and (out[:, 4:] == out[:, 4:5]).all()


def test_int8_gemm_largest_sums_and_shared_addend():
    """Every product 2^14 over the longest k: the sum is 2^14 * 131056, just below 2^31."""
    k = 131056
    a = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((8, k), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    one = torch.ones(1, device=DEV) * 2.0 ** -20
    out = int8_gemm(a, w.t(), one)
    exact = reference_int8_gemm(a, w.t(), one)
    assert (out.double() - exact).abs().max() <= 2.0 ** -8 * exact.abs().max()
    base = torch.ones((3, 8), dtype=torch.bfloat16, device=DEV)
    assert int8_gemm(a, w.t(), one, base=base, output=base) is base  # adds in place
    assert (base.double() - exact - 1).abs().max() <= 2.0 ** -8 * (exact.abs().max() + 1)


@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 4096), (7, 1000), (64, 32768), (2, 8200), (300, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_int8(rows, cols, dtype):
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = (torch.randn((rows, cols), generator=gen, device=DEV) * 3).to(dtype)
    x[0, : 4] = torch.tensor([0.5, -0.5, 0.0, -0.0])
    q, s = quantize_int8(x)
    assert q.dtype == INT8 and s.shape == (rows,)
    wanted = x.double().abs().amax(1) / 127
    assert ((s.double() - wanted).abs() <= 2.0 ** -24 * wanted).all()
    quotient = x.double() / s.double()[:, None]
    # half a step, and what the quotient's rounding to fp32 moves it by
    assert ((q.double() - quotient).abs() <= 0.5 + 2.0 ** -23 * 127).all() and int(q.abs().max()) == 127
    ref, _ = reference_quantize_int8(x, s[:, None])
    assert torch.equal(ref, q)
    static = torch.tensor([0.011], device=DEV)
    q, s = quantize_int8(x, static)
    assert s is static and torch.equal(q, reference_quantize_int8(x, static)[0])
    tiny = torch.tensor([1e-37], device=DEV)  # quotients past fp32 saturate
    assert torch.equal(quantize_int8(x, tiny)[0], torch.sign(x.float()).mul(127).to(INT8))


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_int8_rows_that_are_no_numbers_stay_none(bad):
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((5, 256), generator=gen, device=DEV).bfloat16()
    x[3, 77] = bad
    x[1] = 0
    q, s = quantize_int8(x)
    assert torch.isnan(s).tolist() == [False, False, False, True, False]
    assert (q[1] == 0).all()
    w = _codes(gen, (24, 256), INT8)
    y = apply_int8_linear(x, w, _scales(gen, 24))
    assert torch.isnan(y).any(1).tolist() == [False, False, False, True, False] and torch.isnan(y[3]).all() and (y[1] == 0).all()
    gate_up = torch.randn((4, 64), generator=gen, device=DEV).half()
    gate_up[2, 40] = bad
    assert torch.isnan(swiglu_dynamic(gate_up, dtype=INT8)[1]).tolist() == [False, False, True, False]


@pytest.mark.parametrize("rows,cols", [(1, 8), (9, 1416), (40, 14336)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_swiglu_dynamic_int8(rows, cols, dtype):
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn((rows, 2 * cols), generator=gen, device=DEV).to(dtype)
    q, s = swiglu_dynamic(x, dtype=INT8)
    gate, up = x.double().chunk(2, 1)
    y = gate * torch.sigmoid(gate) * up
    # silu in fp32: exponential and reciprocal of the hardware, 1 unit each, and three products; the scale's largest value has the same error
    rel = 16 * 2.0 ** -24
    assert ((s.double() - y.abs().amax(1) / 127).abs() <= rel * y.abs().amax(1) / 127 + 1e-37).all()
    assert ((q.double() - y / s.double()[:, None]).abs() <= 0.5 + 127 * 2 * rel).all()
    fp8, s8 = swiglu_dynamic(x)
    assert fp8.dtype == FP8 and torch.allclose(s8 * 448, s * 127, rtol=1e-6)


def test_int8_linear_forms():
    gen = torch.Generator(device=DEV).manual_seed(9)
    layer = torch.nn.Linear(320, 200, device=DEV, dtype=torch.bfloat16)
    q = Int8Linear.from_float(layer)
    x = torch.randn((2, 7, 320), generator=gen, device=DEV).bfloat16()
    y = q(x)
    codes, scales = quantize_int8(x.reshape(14, 320))
    exact = reference_int8_gemm(codes, q.weight.t(), scales, q.weight_scale, q.bias).reshape(2, 7, 200)
    magnitude = _magnitude(codes, q.weight, scales, q.weight_scale).reshape(2, 7, 200)
    _close(y, exact, magnitude, 320, INT8, q.bias.expand(2, 7, 200))
    assert (y.float() - layer(x).float()).abs().max() < 0.05  # two roundings to 8 bits of products of sizes below one
    residual = torch.randn((2, 7, 200), generator=gen, device=DEV).bfloat16()
    both = q(x, residual=residual)
    _close(both, exact - q.bias.double() + (residual + q.bias).double(), magnitude, 320, INT8, residual + q.bias)
    assert torch.equal(q(codes, input_scale=scales), y.reshape(14, 200))
    assert torch.equal(apply_int8_linear(x.transpose(0, 1), q.weight, q.weight_scale, bias=q.bias), y.transpose(0, 1))  # the general way
    scalar = torch.tensor(0.5, device=DEV)
    assert torch.allclose(apply_int8_linear(x, q.weight, q.weight_scale, bias=scalar).float(), apply_int8_linear(x, q.weight, q.weight_scale).float() + 0.5, atol=0.02)
    q.half()
    assert q.weight.dtype == INT8 and q.weight_scale.dtype == torch.float32 and q.bias.dtype == torch.float16
    model = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.Linear(32, 10)).to(DEV, torch.bfloat16)
    assert convert_linear_layers(model, dtype=INT8, skip=("1",)) == 1 and isinstance(model[0], Int8Linear)
    assert model(torch.randn(3, 64, device=DEV).bfloat16()).shape == (3, 10)
    loaded = Int8Linear(torch.zeros_like(q.weight), torch.zeros_like(q.weight_scale), torch.zeros_like(q.bias))
    loaded.load_state_dict(q.state_dict())
    assert torch.equal(loaded(x.half()), q(x.half()))


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,k", [(1024, 512), (1030, 768), (6144, 4096), (2304, 8192), (1028, 14336), (1024, 16384), (1024, 16640), (16384, 8192)])
def test_int8_linear_of_few_rows_is_the_two_calls(m, n, k):
    """The bits of quantize_int8 and int8_gemm, for every form of scale and addend, with rows of zeros, of large values, and of NaN."""
    gen = torch.Generator(device=DEV).manual_seed(m + n)
    w, sw = _codes(gen, (n, k), INT8), _scales(gen, n)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn((m, k), generator=gen, device=DEV).to(dtype)
        x[-1, ::3] *= 100
        bias, residual = torch.randn(n, generator=gen, device=DEV).to(dtype), torch.randn((m, n), generator=gen, device=DEV).to(dtype)
        codes, scales = quantize_int8(x)
        for weight_scale, add in ((sw, None), (sw[:1], bias), (None, residual), (sw, residual)):
            got = apply_int8_linear(x, w, weight_scale, bias=add if add is bias else None, residual=add if add is residual else None)
            assert torch.equal(got, int8_gemm(codes, w.t(), scales, weight_scale, base=add, out_dtype=dtype))
        static = torch.tensor([0.02], device=DEV)
        fixed, _ = quantize_int8(x, static)
        assert torch.equal(apply_int8_linear(x, w, sw, static), int8_gemm(fixed, w.t(), static, sw, out_dtype=dtype))
        x[0] = 0
        got = apply_int8_linear(x, w, sw, bias=bias)
        assert torch.equal(got[0], bias)
        x[m - 1, k - 1] = float("nan") if dtype == torch.bfloat16 else float("inf")
        got = apply_int8_linear(x, w, sw)
        assert got[m - 1].isnan().all() and (m == 1 or got[:m - 1].isfinite().all())


def test_int8_linear_without_rows_and_with_more_scales_than_rows():
    w, s = torch.ones((24, 64), dtype=INT8, device=DEV), torch.ones(24, device=DEV)
    assert apply_int8_linear(torch.empty((0, 64), dtype=torch.bfloat16, device=DEV), w, s).shape == (0, 24)
    y = apply_int8_linear(torch.ones((2, 64), dtype=INT8, device=DEV), w, s, torch.tensor([1.0, 2.0, 99.0], device=DEV))
    assert y.tolist() == [[64.0] * 24, [128.0] * 24]


@pytest.mark.parametrize("size", [3, 40, 200])
def test_grouped_on_another_stream_and_in_a_graph(size):
    """Captured once, replayed with other contents of the same tensors: sizes of groups, rows, codes."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    k, n, experts = 256, 96, 4
    count = size * experts
    a, w, sa, sb = _codes(gen, (count, k), FP8), _codes(gen, (experts, n, k), FP8), _scales(gen, count), _scales(gen, experts, n)
    offsets = torch.arange(0, count + 1, size, dtype=torch.int32, device=DEV)
    rows = torch.randperm(count, generator=gen, device=DEV).int()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows))
    out = torch.empty((count, n), dtype=torch.bfloat16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows, output=out)
    for edges in ([0, 1, 1, 2, count], [0, 0, 0, count, count], [0, count // 2, count // 2 + 1, count - 1, count]):
        offsets.copy_(torch.tensor(edges, dtype=torch.int32))
        rows.copy_(torch.randperm(count, generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets, rows=rows))


def test_int8_gemm_on_two_streams_and_in_two_graphs():
    """k in parts: every call has partial sums and counters of its own, so calls at once, and two graphs replayed at once, do not meet."""
    gen = torch.Generator(device=DEV).manual_seed(15)
    (m, n, k), streams = (65, 256, 16384), [torch.cuda.Stream() for _ in range(2)]
    assert _capi.load().hfrk_int8_gemm_workspace_bytes(m, n, k) > 0
    a, w = [_codes(gen, (m, k), INT8) for _ in streams], [_codes(gen, (n, k), INT8) for _ in streams]
    sa = [_scales(gen, m) for _ in streams]
    want = [int8_gemm(x, y.t(), s) for x, y, s in zip(a, w, sa)]
    torch.cuda.synchronize()
    at_once = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                at_once[i].append(int8_gemm(a[i], w[i].t(), sa[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in at_once[i])
    outs, graphs = [torch.empty_like(x) for x in want], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            int8_gemm(a[i], w[i].t(), sa[i], output=outs[i])
    for turn in range(4):
        for i in range(2):
            a[i].copy_(_codes(gen, (m, k), INT8))
            outs[i].fill_(7.0)
        want = [int8_gemm(x, y.t(), s) for x, y, s in zip(a, w, sa)]
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want)), turn


def test_grouped_rows_past_2_31_bytes():
    """Rows in order that lie further than 2^31 bytes into `a`, and a result further than that."""
    k, count = 16384, 140000
    gen = torch.Generator(device=DEV).manual_seed(8)
    a = torch.zeros((count, k), dtype=INT8, device=DEV)
    a[-300:] = _codes(gen, (300, k), INT8)
    w = _codes(gen, (2, 32, k), INT8)
    sa, sb = _scales(gen, count), _scales(gen, 2, 32)
    offsets = torch.tensor([0, count - 250, count], dtype=torch.int32, device=DEV)
    out = grouped_gemm(a, w.transpose(1, 2), sa, sb, offsets)
    for here, e in ((slice(count - 300, count - 250), 0), (slice(count - 250, count), 1)):
        exact = reference_int8_gemm(a[here], w[e].t(), sa[here], sb[e])
        _close(out[here], exact, _magnitude(a[here], w[e], sa[here], sb[e]), k, INT8)
    assert (out[:-300] == 0).all()


def test_refusals():
    gen = torch.Generator(device=DEV).manual_seed(7)
    a, w, s = _codes(gen, (6, 64), INT8), _codes(gen, (2, 32, 64), INT8), _scales(gen, 6)
    b, offsets = w.transpose(1, 2), torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV)
    sb = _scales(gen, 2, 32)
    for bad in (lambda: grouped_gemm(a, b.to(torch.float32).to(FP8), s, sb, offsets), lambda: grouped_gemm(a.float(), b, s, sb, offsets),
                lambda: grouped_gemm(a, w, s, sb, offsets), lambda: grouped_gemm(a, b, s[:5], sb, offsets), lambda: grouped_gemm(a, b, s, sb[:, :31], offsets),
                lambda: grouped_gemm(a, b, s, sb.double(), offsets), lambda: grouped_gemm(a, b, s, sb, offsets.long()), lambda: grouped_gemm(a, b, s, sb, offsets[:2]),
                lambda: grouped_gemm(a, b, s, sb, offsets.cpu()), lambda: grouped_gemm(a, b, s, sb, offsets, rows=torch.zeros(6, device=DEV)),
                lambda: grouped_gemm(a[:, :24], b[:, :24], s, sb, offsets), lambda: grouped_gemm(a[:, :56].contiguous(), b[:, :56], s, sb, offsets),
                lambda: grouped_gemm(a, b, s, sb, offsets, out_dtype=torch.float32),
                lambda: grouped_gemm(a, b, s, sb, offsets, output=torch.empty((5, 32), device=DEV, dtype=torch.half)),
                lambda: int8_gemm(a, w[0], s), lambda: int8_gemm(a, w[0].t(), s, base=torch.zeros(32, device=DEV)), lambda: int8_gemm(a, w[0].t(), s.half()),
                lambda: int8_gemm(a[:, :40].contiguous(), w[0, :, :40].t(), s), lambda: int8_gemm(a, w[0].t().cpu(), s),
                lambda: quantize_int8(torch.zeros((2, 12), device=DEV).half()), lambda: quantize_int8(torch.zeros((2, 16), device=DEV)),
                lambda: swiglu_dynamic(torch.zeros((2, 24), device=DEV).half(), dtype=INT8), lambda: swiglu_dynamic(torch.zeros((2, 32), device=DEV).half(), dtype=torch.uint8)):
        with pytest.raises((AssertionError, RuntimeError)):
            bad()
    memory = torch.zeros(6 * 64 + 6 * 32 * 2, dtype=torch.uint8, device=DEV)
    inside = memory[: 6 * 64].view(INT8).view(6, 64)
    with pytest.raises(RuntimeError, match="share"):
        grouped_gemm(inside, b, s, sb, offsets, output=memory[128:128 + 6 * 64].view(torch.bfloat16).view(6, 32))
    with pytest.raises(RuntimeError, match="share"):
        int8_gemm(inside, w[0].t(), s, output=memory[128:128 + 6 * 64].view(torch.bfloat16).view(6, 32))
    base = torch.zeros(7 * 32, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="base"):
        int8_gemm(a, w[0].t(), s, base=base[:192].view(6, 32), output=base[32:].view(6, 32))
    with pytest.raises(RuntimeError):
        torch.ops._HFRK_C.int8_gemm(a[:, 8:56].contiguous(), w[0, :, 8:56].t(), torch.empty((6, 32), device=DEV, dtype=torch.half), None, s, None)


def test_gradients_are_not_recorded_and_no_tensor_is_changed():
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn((4, 64), generator=gen, device=DEV).bfloat16().requires_grad_()
    w, s = _codes(gen, (16, 64), INT8), _scales(gen, 16)
    y = apply_int8_linear(x, w, s)
    assert not y.requires_grad and hf_rocm_kernels.quantize_int8(x)[0].dtype == INT8


def test_traced_int8_linear_equals_the_eager_layer():
    torch.manual_seed(1)
    layer = Int8Linear.from_float(torch.nn.Linear(1024, 1536, bias=True).to(torch.bfloat16).cuda())
    traced = torch.compile(layer, backend="aot_eager", fullgraph=True)
    for rows in (1, 8, 8, 70):
        x = torch.randn(rows, 1024, device=DEV).to(torch.bfloat16)
        assert torch.equal(traced(x), layer(x)), rows


def test_quantize_int8_of_more_rows_than_one_launch_has():
    """2^26 + 5 rows of a wave each: more threads than the runtime counts."""
    rows = (1 << 26) + 5
    x = torch.full((rows, 8), 127.0, dtype=torch.bfloat16, device=DEV)
    x[-7:] = torch.arange(7, device=DEV, dtype=torch.float32).bfloat16()[:, None]
    codes, scales = quantize_int8(x)
    assert (codes[:-7] == 127).all() and (scales[:-7] == 1.0).all()
    want, want_scales = reference_quantize_int8(x[-7:])
    assert torch.equal(codes[-7:], want) and torch.equal(scales[-7:], want_scales)
