"""Static int8 scales below 2^-126, whose reciprocal is no fp32 number: zeros stay zeros, and codes are quotients as with any other scale."""
import pytest
import torch

from hf_rocm_kernels import quantize_int8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -127, 2.0 ** -128, 3e-39, 1e-40, 2.0 ** -149])
def test_small_static_scales(dtype, scale):
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((5, 264), generator=gen, device=DEV, dtype=torch.float64)
    x[1] *= 60 * scale
    x[2] *= 1e-40
    x[3] = 0.0
    x[4, ::2] = float("inf")
    x[4, 1::2] = -float("inf")
    x = x.to(dtype)
    static = torch.tensor([scale], device=DEV)
    codes, back = quantize_int8(x, static)
    assert back is static
    quotient = (x.double() / static.double()).clamp(-127, 127)
    # half a step, and what the quotient's rounding to fp32 moves it by
    assert ((codes.double() - quotient).abs() <= 0.5 + 2.0 ** -23 * 127).all()
    assert (codes[x == 0] == 0).all()


@pytest.mark.parametrize("scale", [-0.02, -1e20, -3e-39])
def test_scales_below_zero_turn_the_codes(scale):
    """No scale that a checkpoint has; its quotients have codes all the same."""
    x = torch.tensor([[1.0, -2.0, 0.0, 1e20, -3e22, 3e-39, -2e-37, 0.5]], device=DEV, dtype=torch.bfloat16)
    static = torch.tensor([scale], device=DEV)
    codes, _ = quantize_int8(x, static)
    quotient = (x.double() / static.double()).clamp(-127, 127)
    assert ((codes.double() - quotient).abs() <= 0.5 + 2.0 ** -23 * 127).all()
