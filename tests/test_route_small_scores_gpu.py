"""Renormalised weights of choices whose scores are smaller than fp32 holds: every kernel of the router against the plain form in 64 bits."""
import pytest
import torch

from hf_rocm_kernels import route_experts
from hf_rocm_kernels.operators.experts import reference_route_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _logits(tokens, experts, dtype):
    gen = torch.Generator(device=DEV).manual_seed(tokens + experts)
    logits = torch.randn((tokens, experts), generator=gen, device=DEV) * 3
    logits[0] -= 120                     # every choice below what fp32 holds
    logits[1] -= 92                      # about its end
    logits[2, 2:] -= 100                 # two choices far above the others
    logits[3] = torch.linspace(-70, -150, experts, device=DEV)
    logits[4] -= 1e30                    # all the same in fp32
    logits[5, 1:] = torch.finfo(dtype).min
    return logits.to(dtype)


def _check(route, logits, top, rows, **options):
    weights, experts, _, _, _ = reference_route_experts(logits[:rows], top, **{k: (v.cpu() if torch.is_tensor(v) else v) for k, v in options.items()})
    assert torch.equal(route.experts[:rows].cpu(), experts)
    # An exponential's argument, a difference below 128, is rounded by half a step, 2^-18; exponentials, sums of up to 6, products and divisions are off
    # by less than 2^-20 together.  A choice 87 and more below the largest is smaller than 1e-37 of the factor, where fp32's steps are no longer relative
    assert ((route.weights[:rows].cpu().double() - weights).abs() <= 2.0 ** -17 * weights + 1.5 * 1e-37).all()
    total = route.weights.double().sum(1)
    assert ((total - 1.5).abs() <= 1.5 * 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts", [(7, 70), (200, 70), (2100, 70), (2100, 300)])
def test_sigmoid_scores(tokens, experts, dtype):
    logits = _logits(tokens, experts, dtype)
    _check(route_experts(logits, 6, scoring="sigmoid", factor=1.5), logits, 6, 7, scoring="sigmoid", factor=1.5)
    bias = torch.zeros(experts, device=DEV)
    bias[::3] = 2.0  # choices not in the order of their scores
    _check(route_experts(logits, 6, bias=bias, scoring="sigmoid", factor=1.5), logits, 6, 7, bias=bias, scoring="sigmoid", factor=1.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts", [(7, 70), (200, 70), (2100, 70), (2100, 300)])
def test_softmax_scores_of_choices_that_a_bias_makes(tokens, experts, dtype):
    """The bias passes over the experts that have the softmax."""
    logits = _logits(tokens, experts, dtype)
    logits[:, 0] = 40.0
    bias = torch.zeros(experts, device=DEV)
    bias[10:] = 2.0
    _check(route_experts(logits, 6, bias=bias, factor=1.5), logits, 6, 7, bias=bias, factor=1.5)


def test_scores_that_are_not_renormalised_are_what_fp32_holds():
    logits = _logits(7, 70, torch.float32)
    route = route_experts(logits, 6, scoring="sigmoid", renormalize=False)
    weights = reference_route_experts(logits, 6, scoring="sigmoid", renormalize=False)[0]
    # 1 / (1 + e^-x): the exponential within a step (its argument is exact), a sum, a division
    assert ((route.weights.cpu().double() - weights).abs() <= 2.0 ** -21 * weights + 1e-37).all()
