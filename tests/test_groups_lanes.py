"""The router, the experts' sum, groups of few rows and the search for a group's tile from their own sources, lane by lane on the CPU, against 64 bits, with every
tensor flush with pages that nothing may touch: in front of it in one run, behind it in the other.  No GPU."""
import math
import random

import pytest
import torch

from hf_rocm_kernels.operators.experts import reference_combine_experts, reference_route_experts
from hf_rocm_kernels.operators.grouped_gemm import reference_grouped_gemm
from oracle import lane_run_groups as lanes
from test_grouped_gemm_gpu import FP8, INT8, _close

EXPERTS = [1, 2, 63, 64, 65, 128, 129, 200, 512]  # one, two and eight experts a lane, filled and not


def _offsets(experts, count, rng, whole):
    edges = sorted(rng.choice((rng.randint(0, count), 0, count, count // 2)) for _ in range(experts + 1))
    return ([0] + edges[1:-1] + [count]) if whole else edges


@pytest.mark.parametrize("bm", [16, 128, 256])
@pytest.mark.parametrize("experts", EXPERTS)
def test_every_tile_of_every_group_is_found_once(experts, bm):
    rng = random.Random(experts + bm)
    for count, tiles_n, whole in ((1, 1, True), (5, 3, True), (300, 2, False), (1000, 3, True)):
        edges = _offsets(experts, count, rng, whole)
        found = lanes.find_tiles(torch.tensor(edges, dtype=torch.int32), count, bm, tiles_n).tolist()
        sizes = [edges[e + 1] - edges[e] for e in range(experts)]
        wanted = sorted((e, edges[e], size, tile, -(-size // bm)) for e, size in enumerate(sizes) for tile in range(-(-size // bm) * tiles_n))
        assert sorted(tuple(t) for t in found if t[0] >= 0) == wanted, (count, edges)


def test_each_xcd_has_neighbouring_tiles():
    """Workgroups go to the eight XCDs in turn: each has one range of the tiles in the order of the experts."""
    found = lanes.find_tiles(torch.tensor([0, 500, 500, 700, 1000], dtype=torch.int32), 1000, 16, 3).tolist()
    order, first = [], {}
    for e, size in ((0, 500), (2, 200), (3, 300)):
        order += [(e, tile) for tile in range(-(-size // 16) * 3)]
    number = {t: i for i, t in enumerate(order)}
    for x in range(8):
        mine = [number[t[0], t[3]] for t in found[x::8] if t[0] >= 0]
        assert mine == list(range(mine[0], mine[0] + len(mine))) and abs(len(mine) - len(order) / 8) < 1
        first[x] = mine[0]
    assert list(first.values()) == sorted(first.values())


@pytest.mark.parametrize("offsets", [[5, 3, 900, -7], [0, 40, 0, 40], [-(1 << 31), (1 << 31) - 1, 0, 12], [99, 98, 97, 96], [40, 0, 40, 0]])
def test_offsets_that_are_none_lead_to_rows_that_are_there(offsets):
    for bm in (16, 128):
        for e, first, rows, tile, tiles_m in lanes.find_tiles(torch.tensor(offsets, dtype=torch.int32), 40, bm, 3).tolist():
            assert e < 0 or (0 <= e < 3 and 0 <= first and rows > 0 and first + rows <= 40 and 0 <= tile < tiles_m * 3 and tiles_m == -(-rows // bm))


def _route(logits, top, **options):
    """Both runs; the same bits whatever lay in the results and the workspace, and what 64 bits give."""
    route, again = (lanes.route(logits, top, at_end=end, noise=0xff if end else 0x3f, **options) for end in (True, False))
    assert all(torch.equal(x.view(torch.int32), y.view(torch.int32)) for x, y in zip(route, again))
    wanted = reference_route_experts(logits, top, **options)
    for got, want in zip(route[1:], wanted[1:]):
        assert torch.equal(got, want)
    weights, exact = route[0].double(), wanted[0]
    assert torch.equal(torch.isnan(weights), torch.isnan(exact))
    fine = ~torch.isnan(exact)
    # an exponential's argument, a difference below 128, is rounded by half a step, 2^-18; exponentials, sums of up to 32 choices and 512 scores along
    # chains of up to 20, products and divisions are off by less than 2^-19 together; below 1e-37 fp32's steps are no longer relative
    assert ((weights - exact).abs()[fine] <= 2.0 ** -17 * exact.abs()[fine] + 2e-37).all()
    return route


_SIZES = [(1, 1, 1), (3, 5, 5), (17, 8, 2), (64, 60, 4), (65, 64, 6), (40, 512, 8), (70, 300, 8), (100, 65, 32), (30, 130, 17), (130, 256, 10)]


@pytest.mark.parametrize("dtype,tokens,experts,top", [(dtype, *size) for dtype in (torch.bfloat16, torch.float16, torch.float32) for size in _SIZES]
                         + [(torch.bfloat16, 2049, 4, 4), (torch.float32, 2050, 129, 3), (torch.float16, 2051, 70, 17)])
def test_route(dtype, tokens, experts, top):
    gen = torch.Generator().manual_seed(tokens)
    logits = (2 * torch.randn((tokens, experts + 3), generator=gen)).to(dtype)[:, 1:experts + 1] if tokens % 2 else (2 * torch.randn((tokens, experts), generator=gen)).to(dtype)
    bias, mask = 0.1 * torch.randn(experts, generator=gen), torch.rand(tokens, generator=gen) < 0.8
    _route(logits, top)
    _route(logits, top, bias=bias, scoring="sigmoid", factor=2.5, mask=mask)
    if tokens < 2000:
        _route(logits, top, bias=bias, renormalize=False, mask=mask)
        _route(logits, top, scoring="sigmoid", renormalize=False)


def _extreme(tokens, experts):
    logits = 3 * torch.randn((tokens, experts), generator=torch.Generator().manual_seed(experts))
    logits[0] = -math.inf
    logits[1, 2:] = -math.inf
    logits[2, 5] = math.nan
    logits[3, 6] = math.inf
    logits[4] = math.inf
    logits[5] -= 120
    logits[6] = torch.linspace(-70, -150, experts)
    logits[7, 2:] -= 100
    logits[8] -= 1e30
    logits[9, 1:] = torch.finfo(torch.float32).min
    logits[10] = 0.0
    return logits


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts", [(11, 70), (11, 300), (80, 70), (2049, 70)])
def test_route_of_extreme_logits(tokens, experts, scoring):
    """Nothing left, NaN, infinities, scores below fp32's range, ties; a bias that passes over the largest scores, and ones that are infinite or none."""
    logits = _extreme(tokens, experts)
    _route(logits, 4, scoring=scoring)
    passing = torch.zeros(experts)
    passing[10:] = 2.0
    _route(logits, 6, scoring=scoring, bias=passing)
    odd = passing.clone()
    odd[20], odd[21], odd[22] = -math.inf, math.nan, math.inf
    _route(logits, 6, scoring=scoring, bias=odd, factor=0.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [20, 2100])
def test_route_with_a_bias_that_32_bits_cannot_tell(tokens, scoring):
    logits = torch.randn((tokens, 96), generator=torch.Generator().manual_seed(2)) * 2.0 ** -14
    _route(logits, 6, bias=torch.full((96,), 4.0), scoring=scoring)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,top,cols", [(1, 1, 1), (5, 8, 2048), (3, 2, 7), (33, 6, 264), (2, 32, 4104), (7, 3, 2049)])
def test_combine(dtype, tokens, top, cols):
    gen = torch.Generator().manual_seed(cols)
    y = torch.randn((tokens * top, cols), generator=gen).to(dtype)
    places = torch.randperm(tokens * top, generator=gen).int().reshape(tokens, top)
    places[0, 0], places[-1, -1] = -1, tokens * top
    weights, base = torch.rand((tokens, top), generator=gen), torch.randn((tokens, cols), generator=gen).to(dtype)
    for add in (None, base):
        out, again = (lanes.combine(y, weights, places, base=add, at_end=end) for end in (True, False))
        assert torch.equal(out, again)
        exact = reference_combine_experts(y, weights, places, add)
        magnitude = reference_combine_experts(y.abs(), weights, places, None if add is None else add.abs())
        # one rounding to 16 bits; top products and sums in fp32
        bound = torch.finfo(dtype).eps / 2 * (exact.abs() + 1e-4 * magnitude) + (top + 2) * 2.0 ** -24 * magnitude + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert ((out.double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("codes", [FP8, INT8])
@pytest.mark.parametrize("sizes,k,n", [([1], 16, 1), ([1, 0, 2], 48, 7), ([0, 0, 3], 64, 16), ([3, 1, 17, 0, 5], 144, 40), ([2] * 70, 32, 24), ([0] * 130 + [9, 1], 272, 33),
                                       ([20, 0, 1], 1040, 72), ([1, 2, 0, 3], 2064, 130)])
def test_groups_of_few_rows(codes, sizes, k, n):
    """In order and picked, numbers that are no row among them; rows of no group in front and behind; scales a channel, an expert, or one for all rows."""
    gen = torch.Generator().manual_seed(k + n)
    experts, front, behind = len(sizes), 2, 1
    count = sum(sizes) + front + behind
    while count // min(experts, count) > 10:  # (the kernel of few rows)
        sizes, experts = sizes + [0], experts + 1
    offsets = torch.tensor([front + sum(sizes[:e]) for e in range(experts + 1)], dtype=torch.int32)

    def draw(*shape):
        if codes == INT8:
            return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8)
        return (60 * torch.randn(shape, generator=gen)).clamp(-448, 448).to(FP8)

    weight = draw(experts, n, k + 16)[:, :, :k] if n % 2 else draw(experts, n, k)
    for rows, sb in ((None, 0.01 * torch.rand((experts, n), generator=gen)), ("picked", 0.01 * torch.rand(experts, generator=gen)), ("picked", None)):
        a = draw(count if rows is None else 5, k)
        sa = 0.01 * torch.rand(a.size(0) if sb is not None else 1, generator=gen)
        if rows is not None:
            rows = torch.randint(0, 5, (count,), generator=gen, dtype=torch.int32)
            rows[front], rows[-2 if count > 4 else 0] = 5, -1
        out, again = (lanes.grouped(a, weight, sa, sb, offsets, rows, torch.full((count, n), 7.0, dtype=torch.bfloat16), at_end=end) for end in (True, False))
        assert torch.equal(out, again)
        assert (out[:front] == 7.0).all() and (out[count - behind:] == 7.0).all()
        here = slice(front, count - behind)

        def exact(a, weight):
            return reference_grouped_gemm(a, weight.transpose(1, 2), sa.expand(a.size(0)), sb, offsets, rows=rows)[here]

        _close(out[here], exact(a, weight), exact(a.float().abs(), weight.float().abs()), k, codes)
