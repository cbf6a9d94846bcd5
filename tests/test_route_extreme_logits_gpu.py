"""The router on logits of plus infinity: every kernel of it, with a bias and without, against the plain form in 64 bits."""
import math

import pytest
import torch

from hf_rocm_kernels import route_experts
from hf_rocm_kernels.operators.experts import reference_route_experts

DEV = "cuda"


def _check(route, logits, top, first, **options):
    """Rows up to `first`, which hold what is tested, and some others against the plain form."""
    weights, experts, _, _, _ = reference_route_experts(logits[:first], top, **{k: (v.cpu() if torch.is_tensor(v) else v) for k, v in options.items()})
    assert torch.equal(route.experts[:first].cpu(), experts)
    got = route.weights[:first].cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(weights))
    fine = ~torch.isnan(weights)
    # an exponential's argument, a difference below 128, is rounded by half a step, 2^-18; exponentials, sums of 6, products and divisions are
    # off by less than 2^-20 together.  Below 1e-37 the result itself leaves fp32's range
    assert ((got - weights).abs()[fine] <= 2.0 ** -17 * weights.abs()[fine] + 1e-37).all()


def test_plain_form_of_rows_with_plus_infinity():
    logits = torch.randn((3, 8))
    logits[1, 5] = math.inf
    for bias in (None, torch.zeros(8)):
        weights = reference_route_experts(logits, 2, bias=bias)[0]
        assert torch.isnan(weights[1]).all() and torch.isfinite(weights[[0, 2]]).all()
        weights, experts = reference_route_experts(logits, 2, bias=bias, scoring="sigmoid")[:2]
        assert torch.isfinite(weights).all() and int(experts[1, 0]) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts", [(6, 70), (200, 70), (2100, 70), (2100, 300)])
def test_plus_infinity(tokens, experts, dtype):
    """Softmax: the row's scores are none, so its weights are none, with a bias as without one; sigmoid: a score of 1."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    logits = torch.randn((tokens, experts), generator=gen, device=DEV).to(dtype)
    logits[0, 3] = math.inf
    logits[1] = math.inf
    logits[2, 1:] = -math.inf
    logits[2, 0] = math.inf
    logits[3, 5], logits[3, 6] = math.inf, math.nan
    mask = torch.ones(tokens, dtype=torch.bool, device=DEV)
    mask[5] = False
    logits[5, 2] = math.inf
    for bias in (None, 0.1 * torch.randn(experts, generator=gen, device=DEV)):
        for scoring in ("softmax", "sigmoid"):
            for renormalize in (True, False):
                options = dict(bias=bias, scoring=scoring, renormalize=renormalize, mask=mask)
                route = route_experts(logits, 4, **options)
                _check(route, logits, 4, 6, **{**options, "mask": mask[:6]})
                none = torch.isnan(route.weights).all(1)
                assert none[:6].tolist() == ([True] * 4 if scoring == "softmax" else [False, False, False, True]) + [False, False]
                assert not torch.isnan(route.weights[4:]).any() and (route.weights[5] == 0).all()
