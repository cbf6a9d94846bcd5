"""The kernels of attention and append from their own sources, lane by lane on the CPU, against float64, with every tensor flush with pages that nothing
may touch: in front of it in one run, behind it in the other.  No GPU."""
import math
import random
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from hf_rocm_kernels import _capi, rotary_frequencies
from hf_rocm_kernels.operators.append_kv import reference_append_kv
from oracle import attention as oracle
from oracle import lane_run
from test_tree_attention_gpu import FP8, LONG, TYPES, Step, check_small_weights, minus_infinities, small_weights

BOTH_ENDS = (True, False)


def attend(step, at_end, **more):
    call = dict(query=step.query, key_cache=step.key, value_cache=step.value, page_table=step.table, lengths=torch.tensor(step.lengths, dtype=torch.int32),
                starts=step.starts, mask=step.mask, key_scale=step.key_scale, value_scale=step.value_scale)
    return lane_run.attention(**{**call, **more}, at_end=at_end)


def run(step, out_scale=None):
    """Both runs, side by side: right values, rows of nobody left alone, and the same bits whatever the workspace held."""
    scale = None if out_scale is None else torch.tensor([out_scale])

    def one(at_end):
        out = torch.full(step.query.shape, 7.0).to(step.dtype if scale is None else FP8)
        return attend(step, at_end, output=out, out_scale=scale, noise=0xff if at_end else 0x3f)

    with ThreadPoolExecutor(2) as pool:
        results = list(pool.map(one, BOTH_ENDS))
    assert torch.equal(*(r.contiguous().view(torch.uint8) for r in results))
    got = results[0]
    step.check(got.float() if out_scale else got, out_scale=None if out_scale is None else float(torch.tensor(out_scale)))
    assert (got[sum(step.counts):].float() == 7.0).all()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("head_dim", [16, 80, 128, 256])
def test_few_rows(dtype, cache, head_dim):
    run(Step([1, 7, 9, 31, 33, 129, 0, 300], [1] * 8, 8, 2, head_dim, 24, dtype, cache, uniform=True, seed=head_dim))
    run(Step([41, 70, 3], [3, 12, 0], 6, 3, head_dim, 8, dtype, cache, layout="heads", tree="full", seed=head_dim, extra=1))


@pytest.mark.parametrize("dtype,cache,head_dim", [(torch.float16, None, 64), (torch.bfloat16, FP8, 96), (torch.float16, FP8, 256), (torch.bfloat16, None, 144)])
@pytest.mark.parametrize("counts", [[33, 0, 40], [70, 1]])
@pytest.mark.parametrize("tree", [None, "full"])
def test_many_rows(dtype, cache, head_dim, counts, tree):
    """128 and (70 tokens of four heads, up to 128 columns) 256 rows a block."""
    lengths = [n + 37 * (i + 1) for i, n in enumerate(counts)]
    lengths[0] = counts[0]
    step = Step(lengths, counts, 8, 2, head_dim, 16, dtype, cache, tree=tree, seed=sum(counts), extra=2, places=LONG)
    if tree:
        step.mask[1] = False
    run(step)


@pytest.mark.parametrize("heads,kv_heads,counts,places", [(4, 1, [1], 0), (8, 2, [2, 70], 0), (8, 2, [40, 90], LONG), (64, 1, [70], LONG)])
def test_rows_split_between_workgroups(heads, kv_heads, counts, places):
    """Parts joined by a workgroup, a wave or a group of lanes a row (4 to 4480 rows)."""
    run(Step([700 - 100 * i for i in range(len(counts))], counts, heads, kv_heads, 64, 32, torch.float16, seed=3, places=places))


@pytest.mark.parametrize("heads,places", [(4, 0), (32, LONG)])
def test_pages_that_are_missing(heads, places):
    step = Step([3, 90, 60, 50], [6, 2, 2, 4], heads, 2, 64, 16, seed=2, places=places)
    step.table[1, 2], step.table[2, :], step.table[3, 0] = -1, 10 ** 6, -2147483648
    step.lengths[3] = 10 ** 9 if places == 0 else 64
    run(step)


@pytest.mark.parametrize("heads,places", [(4, 0), (32, LONG)])
def test_starts_that_go_back(heads, places):
    """Rows that mean nothing, but no access outside."""
    step = Step([300] * 12, [3] * 12, heads, 2, 64, 16, places=places)
    step.starts = torch.tensor([0 if i % 2 == 0 else 36 for i in range(13)], dtype=torch.int32)
    for at_end in BOTH_ENDS:
        attend(step, at_end)


def test_more_sequences_than_lanes_and_fp8_results():
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 3, (70,), generator=g).tolist()
    run(Step([n + 5 * i % 40 for i, n in enumerate(counts)], counts, 4, 2, 64, 16, torch.float16, seed=1))
    run(Step([200, 20], [2, 5], 8, 2, 128, 16, torch.bfloat16, FP8, seed=4), out_scale=0.004)


@pytest.mark.parametrize("seed", range(5))
def test_drawn(seed):
    r = random.Random(seed)
    for _ in range(3):
        dtype, cache = r.choice(TYPES)
        kv_heads, group, seqs = r.choice([1, 2, 3]), r.choice([1, 2, 5, 7, 17]), r.choice([1, 2, 5])
        head_dim = r.choice([16, 48, 64, 112, 144] if cache == FP8 else [16, 24, 40, 72, 104, 144])
        counts = [r.randint(0, r.choice([1, 2, 9, 20])) for _ in range(seqs)]
        counts[r.randrange(seqs)] += 1
        lengths = [max(0, n + r.choice([-2, 0, 30, 200, 400])) for n in counts]
        step = Step(lengths, counts, kv_heads * group, kv_heads, head_dim, r.choice([8, 24, 40, 1000]), dtype, cache, r.choice(["tokens", "heads"]),
                    r.choice([None, None, "full", 2, 0]), r.randrange(1000), r.choice([0, 3]), places=r.choice([0, LONG]))
        if r.random() < 0.4:
            step.table[r.randrange(seqs), r.randrange(step.table.size(1))] = r.choice([-1, 10 ** 6])
        run(step)


@pytest.mark.parametrize("counts,front,heads,head_dim,places", [([1, 1], 40, 4, 64, 0), ([3, 2], 0, 4, 16, 0), ([5, 9], 300, 8, 64, 0), ([40, 36], 0, 8, 64, LONG),
                                                                ([40, 70], 100, 8, 64, LONG)])
@pytest.mark.parametrize("tree", [False, True])
def test_scores_of_minus_infinity(counts, front, heads, head_dim, places, tree):
    run(minus_infinities(torch.float16 if tree else torch.bfloat16, counts, front, heads, head_dim, tree, places))


# ---- append -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", [None, FP8])
@pytest.mark.parametrize("layout", ["tokens", "heads"])
@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,rotated,interleaved", [
    (1, 8, 2, 128, 128, False), (6, 35, 5, 96, 48, True), (260, 3, 1, 16, 16, False), (5, 4, 4, 80, 0, False), (3, 3, 1, 36, 20, True), (2, 2, 1, 1024, 512, True)])
def test_append(cache, layout, tokens, heads, kv_heads, head_dim, rotated, interleaved):
    g = torch.Generator().manual_seed(tokens)
    dtype, page, pages = torch.float16, 24, 13
    query, key, value = (torch.randn(tokens, n, head_dim, generator=g).to(dtype) for n in (heads, kv_heads, kv_heads))
    shape = (pages, page, kv_heads, head_dim) if layout == "tokens" else (pages, kv_heads, page, head_dim)
    caches = [torch.zeros(shape).to(cache or dtype) for _ in range(2)]
    if layout == "heads":
        caches = [c.transpose(1, 2) for c in caches]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[0] = pages * page - 1
    if tokens > 4:
        slots[1], slots[3] = -1, pages * page
    scales = dict(key_scale=torch.rand(kv_heads, generator=g) + 0.01, value_scale=torch.tensor([0.01])) if cache else {}
    turn = dict(positions=torch.randint(0, 1000, (tokens,), generator=g), frequencies=rotary_frequencies(rotated, device="cpu")[0], interleaved=interleaved) \
        if rotated else {}
    want = [c.clone() for c in caches]
    reference_append_kv(key, value, *want, slots, query=query if rotated else None, **turn, **scales)
    for at_end in BOTH_ENDS:
        got = [c.clone() for c in caches]
        out = torch.zeros_like(query) if rotated else None
        lane_run.append(key, value, *got, slots, query=query if rotated else None, query_output=out, at_end=at_end, **turn, **scales)
        for mine, theirs in zip(got, want):  # (what a rounding is off by may round to the neighbouring value)
            mine, theirs = mine.float(), theirs.float()
            assert ((mine - theirs).abs() <= theirs.abs() * torch.finfo(cache or dtype).eps + 2.0 ** -9).all() and torch.equal(mine != 0, theirs != 0)
        if rotated:
            turned, size = oracle.rotary(query, turn["positions"], turn["frequencies"], interleaved)
            assert ((out.double() - turned).abs() <= oracle.rotary_tolerance(turned, size, dtype)).all()


def test_an_access_outside_is_seen():
    """The check itself: eight sequences, lengths for four."""
    step = Step([5] * 8, [1] * 8, 4, 2, 64, 16, uniform=True)
    with pytest.raises(AssertionError, match="signal 11"):
        attend(step, True, lengths=torch.full((4,), 5, dtype=torch.int32))


@pytest.mark.parametrize("far", [21.5, 23.5, 24.6, 25.0, 28.0])
@pytest.mark.parametrize("tokens,heads,cache", [(1, 2, None), (3, 8, FP8), (40, 8, None)])
def test_many_small_weights_beside_a_large_one_in_fp16(far, tokens, heads, cache):
    """A first token with a large score and a value of zero, and a flat tail `far` powers of two below it: the tail is the result."""
    length, page = 300, 16
    step = small_weights(far, length, page, tokens, heads, cache or torch.float16, places=LONG if tokens == 40 else 0)
    got = lane_run.attention(*step[0])
    check_small_weights(got, *step[1:])


# ---- memory that tensors share --------------------------------------------------------------------------------------------

def shared_step(layout, tokens=3):
    """(query, key, value, key cache, value cache), views of one projection's output and one cache's memory, in a layout that is in use."""
    rows = torch.arange(tokens * 8 * 16, dtype=torch.float32).remainder(251).to(torch.float16)
    if layout == "grouped":          # [tokens, head, (query, key, value)]
        rows = rows[:tokens * 6 * 16].view(tokens, 2, 3, 16)
        step = rows[:, :, 0], rows[:, :, 1], rows[:, :, 2]
    elif layout == "key and value in turn":
        rows = rows.view(tokens, 8, 16)
        step = rows[:, :4], rows[:, 4::2], rows[:, 5::2]
    else:
        rows = rows.view(tokens, 8, 16)
        step = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    memory = torch.zeros(4 * 8 * 2 * 2 * 16, dtype=torch.float16)
    if layout == "pages in turn":
        both = memory.view(4, 2, 8, 2, 16)
        caches = both[:, 0], both[:, 1]
    elif layout == "heads side by side":
        both = memory.view(4, 8, 4, 16)
        caches = both[:, :, :2], both[:, :, 2:]
    elif layout == "columns side by side":
        both = memory.view(4, 8, 2, 32)
        caches = both[..., :16], both[..., 16:]
    elif layout == "keys by heads, values by tokens":
        both = memory.view(4, 2, 256)
        caches = both[:, 0].view(4, 2, 8, 16).transpose(1, 2), both[:, 1].view(4, 8, 2, 16)
    elif layout == "layers in turn":
        both = memory.view(2, 4, 8, 2, 16)
        caches = both[0], both[1]
    else:
        caches = memory[:1024].view(4, 8, 2, 16), memory[1024:].view(4, 8, 2, 16)
    return (*step, *caches)


SLOTS, TURN = torch.tensor([5, 31, 8]), dict(positions=torch.tensor([1, 7, 30]), frequencies=torch.tensor([0.5] * 8, dtype=torch.float64))


@pytest.mark.parametrize("tokens", [3, 1])
@pytest.mark.parametrize("layout", ["plain", "grouped", "key and value in turn", "pages in turn", "heads side by side", "columns side by side",
                                    "keys by heads, values by tokens", "layers in turn"])
def test_views_of_one_memory_that_lie_between_each_other(layout, tokens):
    query, key, value, *caches = shared_step(layout, tokens)
    turn = dict(positions=TURN["positions"][:tokens], frequencies=TURN["frequencies"])
    want = [c.clone() for c in caches]
    turned = reference_append_kv(key, value, *want, SLOTS[:tokens], query=query, **turn)
    assert lane_run.append_where_they_are(key, value, *caches, SLOTS[:tokens], query=query, query_output=query, **turn) == _capi.SUCCESS
    assert (query.float() - turned.float()).abs().max() <= 0.25 and all((a.float() - b.float()).abs().max() <= 0.25 for a, b in zip(caches, want))


def overlapping(case):
    query, key, value, key_cache, value_cache = shared_step("plain")
    rows = query.as_strided((3, 8, 16), (128, 16, 1), 0)
    memory = key_cache.as_strided((2048,), (1,), 0)
    call = dict(query=query, query_output=query, key=key, value=value, key_cache=key_cache, value_cache=value_cache)
    if case == "in place over a key head":
        call.update(query=rows[:, :5], query_output=rows[:, :5])
    elif case == "in place, the keys themselves":
        call.update(query=key, query_output=key)
    elif case == "in place over a value head of another token":
        call.update(value=rows.as_strided((2, 2, 16), (128, 16, 1), 128), key=key[1:], query=query[:2], query_output=rows.as_strided((2, 4, 16), (128, 16, 1), 64))
        call.update(query=call["query_output"])
    elif case == "an output shifted by a head":
        call.update(query=rows[:, :3], query_output=rows[:, 1:4])
    elif case == "an output whose heads overlap":
        call.update(query_output=torch.zeros(400, dtype=torch.float16).as_strided((3, 4, 16), (64, 8, 1)))
    elif case == "an output whose tokens overlap":
        call.update(query_output=torch.zeros(400, dtype=torch.float16).as_strided((3, 4, 16), (32, 16, 1)))
    elif case == "caches a page apart":
        call.update(key_cache=memory[:1024].view(4, 8, 2, 16), value_cache=memory[256:1280].view(4, 8, 2, 16))
    elif case == "caches a head apart":
        call.update(key_cache=memory.view(4, 8, 4, 16)[:, :, :2], value_cache=memory.view(4, 8, 4, 16)[:, :, 1:3])
    elif case == "caches eight columns apart":
        call.update(key_cache=memory.view(4, 8, 2, 32)[..., :16], value_cache=memory.view(4, 8, 2, 32)[..., 8:24])
    elif case == "one cache":
        call.update(value_cache=key_cache)
    elif case == "places that overlap":
        call.update(key_cache=memory.as_strided((4, 8, 2, 16), (256, 16, 16, 1)))
    elif case == "pages that overlap":
        call.update(value_cache=memory[1024:].as_strided((4, 8, 2, 16), (128, 32, 16, 1)))
    elif case == "a cache and the step":
        call.update(key_cache=rows.as_strided((1, 8, 2, 16), (0, 32, 16, 1), 100))
        call.update(value_cache=value_cache[:1])
    return call


@pytest.mark.parametrize("case", ["in place over a key head", "in place, the keys themselves", "in place over a value head of another token",
                                  "an output shifted by a head", "an output whose heads overlap", "an output whose tokens overlap", "caches a page apart",
                                  "caches a head apart", "caches eight columns apart", "one cache", "places that overlap", "pages that overlap",
                                  "a cache and the step"])
def test_memory_that_is_written_and_used_by_others_is_refused(case):
    call = overlapping(case)
    n = call["key"].size(0)
    assert lane_run.append_where_they_are(**call, slots=SLOTS[:n], positions=TURN["positions"][:n], frequencies=TURN["frequencies"]) == _capi.BAD_SHAPE


def test_what_meets_by_counting_bytes():
    """Drawn views of one buffer: refused where two of a launch's threads use a byte that one of them writes, and, the strides lying within each
    other, nowhere else."""
    r = random.Random(1)
    memory = torch.zeros(4096, dtype=torch.float16)
    refused = 0
    for _ in range(400):
        token, head = r.choice([64, 128, 200]), r.choice([16, 32, 48])
        def view(n):
            return memory.as_strided((r.choice([1, 2, 3]), n, 16), (token, head, 1), r.randrange(0, 256, 8))
        query, output = view(r.choice([1, 2])), view(2)
        output = output[:query.size(0), :query.size(1)]
        query = query[:output.size(0)]
        if (output.size(1) - 1) * head + 16 > token:
            continue
        used = [{int(x) for x in (torch.arange(4096).as_strided(t.shape, t.stride(), t.storage_offset())).flatten()} for t in (query, output)]
        apart = not (used[0] & used[1]) or (query.storage_offset() == output.storage_offset())
        status = lane_run.append_where_they_are(None, None, None, None, None, torch.arange(query.size(0)), TURN["frequencies"], query=query, query_output=output)
        assert status == (_capi.SUCCESS if apart else _capi.BAD_SHAPE)
        refused += not apart
    assert 50 < refused < 350


@pytest.mark.parametrize("head_dim", [16, 18])
def test_fp8_keeps_nan_and_saturates_infinities(head_dim):
    """Caches and results in e4m3fn: no NaN becomes a number.  (Vector and scalar kernel.)"""
    key = torch.zeros(1, 1, head_dim, dtype=torch.float16)
    key[0, 0, :6] = torch.tensor([math.nan, math.inf, -math.inf, 3e4, -math.nan, 449.0])
    caches = [torch.zeros(1, 8, 1, head_dim).to(FP8) for _ in range(2)]
    lane_run.append(key, key, *caches, torch.tensor([3]))
    for c in caches:
        got = c[0, 3, 0].float()
        assert torch.isnan(got[[0, 4]]).all() and torch.equal(got[[1, 2, 3, 5, 6]], torch.tensor([448.0, -448.0, 448.0, 448.0, 0.0]))


@pytest.mark.parametrize("places", [0, LONG])
def test_a_result_in_fp8_keeps_nan(places):
    step = minus_infinities(torch.bfloat16, [40, 40], 0, 8, 64, False, places)
    got = attend(step, True, out_scale=torch.tensor([0.01])).float()
    assert torch.isnan(got[:40]).all() and torch.isfinite(got[40:]).all()
