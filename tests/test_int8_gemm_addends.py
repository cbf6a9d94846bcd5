"""The addend of `int8_gemm`: (m, n) or (n,) as documented; every other shape is refused, whichever way a call goes."""
import pytest
import torch

from hf_rocm_kernels.operators.int8_gemm import int8_gemm, reference_int8_gemm, wrapped

M, N, K = 6, 32, 64
_OTHER_SHAPES = [(), (1,), (M,), (1, M, N), (N, M), (1, M * N), (M * N,), (1, N), (M, 1), (M, N, 1), (2, M // 2, N)]


def _operands(device):
    gen = torch.Generator().manual_seed(0)
    a, w = (torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8).to(device) for shape in ((M, K), (N, K)))
    return a, w.t(), (0.001 + 0.01 * torch.rand(M, generator=gen)).to(device)


@pytest.mark.parametrize("shape", _OTHER_SHAPES)
def test_other_shapes_do_not_reach_the_native_operator(shape, monkeypatch):
    """On the CPU, with the native operator replaced by a recorder: it is not asked, and the checks name the addend."""
    asked = []
    monkeypatch.setattr(wrapped, "runs_now", lambda t: True)
    monkeypatch.setattr(wrapped, "_int8_linear", lambda *args: asked.append(args) or torch.zeros((M, N), dtype=torch.bfloat16))
    a, b, scale = _operands("cpu")
    with pytest.raises(AssertionError, match="base"):
        int8_gemm(a, b, scale, base=torch.ones(shape, dtype=torch.bfloat16))
    assert not asked


@pytest.mark.parametrize("shape", [None, (N,), (M, N)])
def test_documented_shapes_reach_the_native_operator(shape, monkeypatch):
    asked = []
    monkeypatch.setattr(wrapped, "runs_now", lambda t: True)
    monkeypatch.setattr(wrapped, "_int8_linear", lambda *args: asked.append(args) or torch.zeros((M, N), dtype=torch.bfloat16))
    a, b, scale = _operands("cpu")
    base = None if shape is None else torch.ones(shape, dtype=torch.bfloat16)
    int8_gemm(a, b, scale, base=base)
    (_, _, _, _, bias, residual, _), = asked
    assert bias is (base if shape == (N,) else None) and residual is (base if shape == (M, N) else None)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", _OTHER_SHAPES)
def test_other_shapes_are_refused(shape):
    a, b, scale = _operands("cuda")
    base = torch.ones(shape, dtype=torch.bfloat16, device="cuda")
    for output in (None, torch.empty((M, N), dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(AssertionError, match="base"):
            int8_gemm(a, b, scale, base=base, output=output)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(N,), (M, N)])
def test_documented_shapes_are_added(shape):
    a, b, scale = _operands("cuda")
    base = torch.full(shape, 3.0, dtype=torch.bfloat16, device="cuda")
    out = int8_gemm(a, b, scale, base=base)
    exact = reference_int8_gemm(a, b, scale, None, base)
    # one rounding to bfloat16, and in front of it the sum, its scale and the addend in fp32: 3 * 2^-24 of the product's and the addend's size
    bound = 2.0 ** -8 * exact.abs() + 3 * 2.0 ** -24 * 1.01 * ((exact - 3).abs() + 3)
    assert ((out.double() - exact).abs() <= bound).all()
    assert torch.equal(int8_gemm(a, b, scale, base=base, output=torch.empty_like(out)), out)
