"""Rotary positions and the append to a paged cache against float64, at the sizes and layouts where a kernel can go wrong."""
import math

import pytest
import torch

from hf_rocm_kernels import append_kv, rotary, rotary_frequencies
from oracle import attention as oracle

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
BOTH = (torch.bfloat16, torch.float16)


def _heads(g, tokens, heads, head_dim, dtype):
    return torch.randn(tokens, heads, head_dim, generator=g).to(dtype)


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _check_rotated(got, x, positions, frequencies, interleaved, magnitude=1.0):
    want, size = oracle.rotary(x, positions, frequencies, interleaved, magnitude)
    got = got.cpu()
    assert ((got.double() - want).abs() <= oracle.rotary_tolerance(want, size, x.dtype)).all()
    kept = 2 * frequencies.numel()
    assert torch.equal(_bits(got[..., kept:]), _bits(x[..., kept:]))  # copied values keep their bits


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,head_dim,rotated", [
    (1, 40, 128, 128), (1, 1, 16, 16), (5, 3, 128, 64), (7, 37, 80, 32), (2, 9, 96, 96), (3, 5, 64, 48), (257, 2, 128, 128), (300, 3, 256, 32),
    (2, 2, 1024, 1024),                                               # whole 16-byte pieces
    (3, 5, 80, 20), (2, 3, 7, 6), (4, 1, 2, 2), (1, 70, 100, 100), (300, 1, 40, 8), (2, 3, 128, 0)])  # others
def test_rotation(dtype, interleaved, tokens, heads, head_dim, rotated):
    g = torch.Generator().manual_seed(tokens + heads + rotated)
    x = _heads(g, tokens, heads, head_dim, dtype)
    frequencies = rotary_frequencies(rotated, 10000.0, device="cpu")[0] if rotated else torch.empty(0, dtype=torch.float64)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g)
    for p, f in ((positions, frequencies), (positions.int(), frequencies.float())):
        got = rotary(x.cuda(), p.cuda(), f.cuda(), interleaved=interleaved)
        _check_rotated(got, x, p, f, interleaved)


@pytest.mark.parametrize("position", [0, 1, -5, (1 << 24) + 1, (1 << 31) + 12345, 1 << 40])
def test_rotation_far_out(position):
    """A turn is formed in 64 bits: 2^-53 of 2^40 positions at a radian each is 2^-13 of a radian, far positions of less nothing."""
    x = _heads(torch.Generator().manual_seed(3), 1, 2, 128, torch.bfloat16)
    frequencies = rotary_frequencies(128, 500000.0, device="cpu")[0]
    p = torch.tensor([position])
    got = rotary(x.cuda(), p.cuda(), frequencies.cuda(), magnitude=0.75).cpu().double()
    want, size = oracle.rotary(x, p, frequencies, False, 0.75)
    angle = abs(position) * frequencies * 4 * 2.0 ** -53
    assert ((got - want).abs() <= oracle.rotary_tolerance(want, size, x.dtype) + size * torch.cat((angle, angle))).all()


def test_rotation_of_slices_in_place_and_into_others():
    g = torch.Generator().manual_seed(5)
    rows = _heads(g, 9, 14, 128, torch.bfloat16)
    frequencies, positions = rotary_frequencies(64, device="cuda")[0], torch.arange(100, 109, device="cuda")
    want = rotary(rows[:, :10].contiguous().cuda(), positions, frequencies, interleaved=True)
    _check_rotated(want, rows[:, :10], positions.cpu(), frequencies.cpu(), True)
    there = rows.cuda()
    assert rotary(there[:, :10], positions, frequencies, interleaved=True, output=there[:, :10]).data_ptr() == there.data_ptr()
    assert torch.equal(_bits(there[:, :10]), _bits(want)) and torch.equal(_bits(there[:, 10:]), _bits(rows[:, 10:].cuda()))
    wide = torch.zeros(9, 10, 200, dtype=torch.bfloat16, device="cuda")
    rotary(rows.cuda()[:, :10], positions, frequencies, interleaved=True, output=wide[..., 8:136])
    assert torch.equal(_bits(wide[..., 8:136]), _bits(want)) and not wide[..., :8].any() and not wide[..., 136:].any()
    rotary(rows.cuda()[:, :10], positions, frequencies, interleaved=True, output=wide[..., 3:131])  # off every boundary
    assert torch.equal(_bits(wide[..., 3:131]), _bits(want))
    by_heads = rows[:, :10].transpose(0, 1).contiguous().cuda().transpose(0, 1)  # heads outermost
    assert torch.equal(_bits(rotary(by_heads, positions, frequencies, interleaved=True)), _bits(want))


def test_rotation_keeps_infinities_and_nan_where_they_are():
    x = torch.zeros(1, 2, 32, dtype=torch.float16)
    x[0, 0, 3], x[0, 1, 31] = math.inf, math.nan
    got = rotary(x.cuda(), torch.tensor([1], device="cuda"), torch.tensor([0.5] * 8, device="cuda")).cpu()
    assert got[0, 0, 3] == math.inf and got[0, 0, 11] == math.inf and torch.isnan(got[0, 1, 31]) and int(torch.isfinite(got).sum()) == 61


def test_rotation_of_nothing():
    f = torch.ones(4, device="cuda")
    none = torch.empty(0, 3, 16, dtype=torch.float16, device="cuda")
    assert rotary(none, torch.empty(0, dtype=torch.long, device="cuda"), f).shape == (0, 3, 16)
    assert rotary(none.view(3, 0, 16), torch.zeros(3, dtype=torch.long, device="cuda"), f).shape == (3, 0, 16)


# ---- append -------------------------------------------------------------------------------------------------------------

def _caches(g, pages, page, kv_heads, head_dim, dtype, layout):
    if layout == "pair":  # keys and values of a page side by side in one tensor
        both = torch.randn(pages, 2, page, kv_heads, head_dim, generator=g).to(dtype).cuda()
        return both[:, 0], both[:, 1]
    if layout == "heads":
        return tuple(torch.randn(pages, kv_heads, page, head_dim, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    return tuple(torch.randn(pages, page, kv_heads, head_dim, generator=g).to(dtype).cuda() for _ in range(2))


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, FP8), (torch.float16, FP8)])
@pytest.mark.parametrize("layout", ["tokens", "heads", "pair"])
@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,rotated,interleaved", [
    (1, 32, 8, 128, 128, False), (6, 35, 5, 96, 48, True), (300, 4, 2, 64, 64, False), (5, 4, 4, 80, 0, False), (3, 3, 1, 36, 20, True), (9, 6, 3, 24, 24, False)])
def test_append(dtype, cache, layout, tokens, heads, kv_heads, head_dim, rotated, interleaved):
    g = torch.Generator().manual_seed(tokens + head_dim)
    page, pages = 24, 20
    rows = torch.randn(tokens, heads + 2 * kv_heads, head_dim, generator=g).to(dtype)
    query, key, value = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    caches = _caches(g, pages, page, kv_heads, head_dim, cache or dtype, layout)
    before = [c.clone() for c in caches]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[3] = -1, pages * page  # padding
    positions = torch.randint(0, 100000, (tokens,), generator=g)
    frequencies = rotary_frequencies(rotated, device="cpu")[0] if rotated else None
    scales = (torch.rand(kv_heads, generator=g) * 0.02 + 0.004, torch.tensor([0.01])) if cache else (None, None)
    there = rows.cuda()
    q = there[:, :heads]
    turn = dict(positions=positions.cuda(), frequencies=frequencies.cuda(), interleaved=interleaved, query=q, query_output=q) if rotated else {}
    got = append_kv(there[:, heads:heads + kv_heads], there[:, heads + kv_heads:], *caches, slots.cuda() if tokens % 2 else slots.int().cuda(),
                    key_scale=scales[0].cuda() if cache else None, value_scale=scales[1].cuda() if cache else None, **turn)
    torch.cuda.synchronize()
    if rotated:
        assert got.data_ptr() == q.data_ptr()
        _check_rotated(got, query, positions, frequencies, interleaved)
    else:
        assert got is None
    assert torch.equal(_bits(there[:, heads:]), _bits(rows[:, heads:].cuda()))  # the step's keys and values stay
    kept = (slots >= 0) & (slots < pages * page)
    where = slots[kept] // page, slots[kept] % page
    none = torch.zeros_like(key[kept], dtype=torch.float64)
    want_key = oracle.rotary(key, positions, frequencies, interleaved) if rotated else (key.double(), torch.zeros(key.shape, dtype=torch.float64))
    for c, old, (want, size), scale in ((caches[0], before[0], (want_key[0][kept], want_key[1][kept]), scales[0]),
                                        (caches[1], before[1], (value[kept].double(), none), scales[1])):
        c, old = c.cpu(), old.cpu()
        mine = (c.view(torch.uint8)[where].view(c.dtype) if cache else c[where]).double()
        if cache:
            by = scale.double().reshape(1, -1, 1)
            want, size = want / by, size / by
            # a quotient by the reciprocal: two more roundings of 2^-24; saturation at 448 (half a step above it rounds to it too)
            off = want.abs() * (oracle.half_step(FP8) * (1 + 2.0 ** -10) + 2.0 ** -22) + oracle.smallest_step(FP8) + size * 2.0 ** -21
            assert ((mine - want.clamp(-448, 448)).abs() <= off).all()
        elif bool((size > 0).any()):
            assert ((mine - want).abs() <= oracle.rotary_tolerance(want, size, dtype)).all()
        else:
            assert torch.equal(mine, want)
        # nothing else has been touched
        left = torch.ones(c.shape[:2], dtype=torch.bool)
        left[where] = False
        assert torch.equal(c.view(torch.uint8)[left], old.view(torch.uint8)[left]) if cache else torch.equal(_bits(c[left]), _bits(old[left]))


def test_append_saturates_and_fills_the_last_slot():
    key = torch.full((1, 1, 16), 3.0e4, dtype=torch.float16, device="cuda")
    caches = [torch.zeros(2, 8, 1, 16, device="cuda").to(FP8) for _ in range(2)]
    append_kv(key, -key, *caches, torch.tensor([15], device="cuda"))
    for c, x in zip(caches, (448.0, -448.0)):
        c = c.float()
        assert (c[1, 7] == x).all() and int((c != 0).sum()) == 16


def test_append_past_32_bits():
    """Pages so far apart that their offsets in elements need more than 32 bits."""
    memory = torch.zeros(2, 3, 1 << 30, dtype=torch.bfloat16, device="cuda")  # 12 GB
    key_cache, value_cache = (memory[i].view(-1).as_strided((3, 16, 2, 64), (1 << 30, 128, 64, 1)) for i in range(2))
    g = torch.Generator().manual_seed(1)
    key, value = (torch.randn(2, 2, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    append_kv(key, value, key_cache, value_cache, torch.tensor([2 * 16 + 15, 16], device="cuda"))
    assert torch.equal(key_cache[2, 15], key[0]) and torch.equal(value_cache[1, 0], value[1]) and torch.equal(value_cache[2, 15], value[0])


def test_append_on_another_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(8)
    rows = torch.randn(4, 12, 128, generator=g).to(torch.bfloat16).cuda()
    frequencies = rotary_frequencies(128)[0]
    slots, positions = torch.zeros(4, dtype=torch.long, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    caches = [torch.zeros(8, 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    eager = [torch.zeros_like(c) for c in caches]

    def step(to):
        return append_kv(rows[:, 8:10], rows[:, 10:], *to, slots, positions, frequencies, query=rows[:, :8])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([torch.zeros_like(c) for c in caches])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned = step(caches)
    for n in range(4):
        slots.copy_(torch.tensor([n, 20 + n, 127 - n, -1]))
        positions.copy_(torch.tensor([5 * n, 7, 100000 + n, 3]))
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(turned, want) and all(torch.equal(a, b) for a, b in zip(caches, eager))


def test_whole_calls_and_general_ones_give_the_same_bits(monkeypatch):
    from hf_rocm_kernels.operators.append_kv import wrapped as append_wrapped
    from hf_rocm_kernels.operators.rotary import wrapped as rotary_wrapped
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(7, 12, 64, generator=g).to(torch.float16).cuda()
    positions, frequencies = torch.arange(7, device="cuda"), rotary_frequencies(64)[0]

    def calls():
        caches = [torch.zeros(2, 16, 2, 64, dtype=torch.float16, device="cuda") for _ in range(4)]
        with_query = append_kv(rows[:, 8:10], rows[:, 10:], *caches[:2], positions, positions, frequencies, query=rows[:, :8])
        assert append_kv(rows[:, 8:10], rows[:, 10:], *caches[2:], positions) is None
        return [rotary(rows, positions, frequencies), with_query, *caches]

    got = calls()
    monkeypatch.setattr(rotary_wrapped, "_rotary_new", lambda *args: None)
    monkeypatch.setattr(append_wrapped, "_append_kv_new", lambda *args: (False, None))
    assert all(torch.equal(a, b) for a, b in zip(got, calls()))


def test_refused_on_the_device():
    """What the checks in front do not see: results that overlap their inputs, and devices."""
    rows = torch.zeros(3, 6, 64, dtype=torch.bfloat16, device="cuda")
    positions, frequencies = torch.zeros(3, dtype=torch.long, device="cuda"), torch.ones(32, device="cuda")
    with pytest.raises(RuntimeError, match="apart"):
        rotary(rows[:, :4], positions, frequencies, output=rows[:, 1:5])
    with pytest.raises(RuntimeError, match="apart"):
        rotary(rows, positions, frequencies, output=rows[:, :1].expand(3, 6, 64))
    with pytest.raises(AssertionError, match="positions.device"):
        rotary(rows, positions.cpu(), frequencies)
    cache = torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="same memory"):
        append_kv(rows[:, 2:4], rows[:, 4:], cache, cache, positions)
    with pytest.raises(RuntimeError, match="apart"):
        append_kv(cache[:, 0], rows[:, 4:], cache, torch.zeros_like(cache), positions)
    with pytest.raises(RuntimeError, match="query_output"):
        append_kv(rows[:, 2:4], rows[:, 4:], cache, torch.zeros_like(cache), positions, positions, frequencies, query=rows[:, :2].clone(),
                  query_output=rows[:, 3:5])


def test_shared_memory_is_refused_on_the_device():
    rows = torch.zeros(3, 8, 64, dtype=torch.bfloat16, device="cuda")
    memory = torch.zeros(4, 8, 4, 64, dtype=torch.bfloat16, device="cuda")
    turn = dict(positions=torch.zeros(3, dtype=torch.long, device="cuda"), frequencies=torch.ones(32, device="cuda"))
    slots = torch.arange(3, device="cuda")
    with pytest.raises(RuntimeError, match="query_output must lie apart"):  # a key's head is turned by one thread and read by another
        append_kv(rows[:, 4:6], rows[:, 6:], memory[:, :, :2], memory[:, :, 2:], slots, query=rows[:, :5], query_output=rows[:, :5], **turn)
    with pytest.raises(RuntimeError, match="same memory"):
        append_kv(rows[:, 4:6], rows[:, 6:], memory[:, :, :2], memory[:, :, 1:3], slots)
    with pytest.raises(RuntimeError, match="overlap themselves"):
        append_kv(rows[:, 4:6], rows[:, 6:], memory[:2, :, :2].as_strided((2, 8, 2, 64), (256, 64, 64, 1)), memory[2:, :, :2], slots)
    with pytest.raises(RuntimeError, match="apart"):
        rotary(rows, **turn, output=rows.as_strided((3, 8, 64), (512, 32, 1)))
    # heads in groups of (query, key, value), turned where they are, and caches side by side in a head
    grouped = torch.randn(3, 2, 3, 64, device="cuda").to(torch.bfloat16)
    want = rotary(grouped[:, :, 0].contiguous(), **turn)
    query = grouped[:, :, 0]
    append_kv(grouped[:, :, 1], grouped[:, :, 2], memory[:, :, :2], memory[:, :, 2:], slots, query=query, query_output=query, **turn)
    assert torch.equal(query, want) and torch.equal(memory[0, :3, 2:], grouped[:, :, 2])


def test_more_tokens_than_a_launch_has_workgroups():
    """2^24 workgroups of 256 threads are more than 32 bits count."""
    tokens = (1 << 24) + 5
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = torch.randn(tokens, 3, 2, generator=g, device="cuda").to(torch.float16)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    frequencies = torch.tensor([0.37], dtype=torch.float64, device="cuda")
    memory = torch.zeros(2, 1 << 20, 17, 1, 2, dtype=torch.float16, device="cuda")
    got = append_kv(rows[:, 1:2], rows[:, 2:], memory[0], memory[1], positions, positions, frequencies, query=rows[:, :1])
    some = torch.cat((torch.arange(3), (1 << 23) + torch.arange(-3, 3), (1 << 24) + torch.arange(-3, 5)))
    x = rows[some.cuda()].cpu()
    want, size = oracle.rotary(x[:, :2], some, frequencies.cpu(), False)
    mine = torch.cat((got[some.cuda()].cpu(), memory[0].view(-1, 1, 2)[some.cuda()].cpu()), dim=1)
    assert ((mine.double() - want).abs() <= oracle.rotary_tolerance(want, size, torch.float16)).all()
    assert torch.equal(memory[1].view(-1, 1, 2)[:tokens], rows[:, 2:]) and not memory[:, -1].any()
    assert torch.equal(rotary(rows[:, :1], positions, frequencies), got)


@pytest.mark.parametrize("head_dim", [16, 18])
def test_append_in_fp8_keeps_nan_and_saturates_infinities(head_dim):
    key = torch.zeros(1, 1, head_dim, dtype=torch.float16, device="cuda")
    key[0, 0, :6] = torch.tensor([math.nan, math.inf, -math.inf, 3e4, -math.nan, 449.0])
    caches = [torch.zeros(1, 8, 1, head_dim, device="cuda").to(FP8) for _ in range(2)]
    append_kv(key, key, *caches, torch.tensor([3], device="cuda"))
    for c in caches:
        got = c[0, 3, 0].float().cpu()
        assert torch.isnan(got[[0, 4]]).all() and torch.equal(got[[1, 2, 3, 5, 6]], torch.tensor([448.0, -448.0, 448.0, 448.0, 0.0]))


def test_a_launch_whose_first_token_is_past_31_bits_of_bytes():
    """Slices of a call that begin 2^30 tokens in, or later: their offsets in bytes need more than 32 bits."""
    tokens = (1 << 30) + (1 << 23) + 5
    x = torch.empty(tokens, 1, 2, dtype=torch.float16, device="cuda")
    some = torch.cat((torch.arange(3), (1 << 30) + torch.arange(-3, 3), tokens + torch.arange(-8, 0)))
    x[some.cuda()] = torch.randn(some.numel(), 1, 2, generator=torch.Generator().manual_seed(1)).to(torch.float16).cuda()
    positions = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    positions[some.cuda()] = torch.arange(some.numel(), dtype=torch.int32, device="cuda")
    frequencies = torch.tensor([0.37], dtype=torch.float64, device="cuda")
    before = x[some.cuda()].cpu()
    assert rotary(x, positions, frequencies, output=x) is x
    _check_rotated(x[some.cuda()], before, torch.arange(some.numel()), frequencies.cpu(), False)
