"""Rotary positions, append and attention without a GPU: refusals (the wrappers' and the C ABI's, which answers before it touches a device), shapes under
fake tensors, frequencies, the Torch forms against the oracle, and the division by the page size."""
import ctypes
import math

import pytest
import torch
from torch._subclasses import FakeTensorMode

import hf_rocm_kernels
from hf_rocm_kernels import _capi, append_kv, rotary, rotary_frequencies, tree_attention
from hf_rocm_kernels.operators.append_kv import reference_append_kv
from hf_rocm_kernels.operators.rotary import reference_rotary
from hf_rocm_kernels.operators.tree_attention import reference_tree_attention
from oracle import attention as oracle

FP8 = torch.float8_e4m3fn
BF16 = torch.bfloat16


# ---- the wrappers -------------------------------------------------------------------------------------------------------

def _rotary_call(**changes):
    call = dict(x=torch.zeros(3, 4, 64, dtype=BF16), positions=torch.zeros(3, dtype=torch.long), frequencies=torch.ones(32, dtype=torch.float64))
    call.update(changes)
    return call


@pytest.mark.parametrize("changes,says", [
    ({}, "cuda"),
    (dict(x=torch.zeros(4, 64, dtype=BF16)), "3 dimensions"),
    (dict(x=torch.zeros(3, 4, 64)), "bfloat16 or torch.float16"),
    (dict(x=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2)), "unit stride"),
    (dict(x=torch.zeros(3, 1, 1040, dtype=BF16)), "1 to 1024"),
    (dict(positions=torch.zeros(4, dtype=torch.long)), "positions.shape"),
    (dict(positions=torch.zeros(3)), "int32 or torch.int64"),
    (dict(positions=torch.zeros(6, dtype=torch.long)[::2]), "contiguous"),
    (dict(frequencies=torch.ones(33)), "at most 32 frequencies"),
    (dict(frequencies=torch.ones(32, dtype=BF16)), "float32 or torch.float64"),
    (dict(output=torch.zeros(3, 4, 64, dtype=torch.float16)), "output like x"),
    (dict(output=torch.zeros(3, 4, 32, dtype=BF16)), "output like x")])
def test_rotary_refuses(changes, says):
    with pytest.raises(AssertionError, match=says):
        rotary(**_rotary_call(**changes))


def _append_call(**changes):
    call = dict(key=torch.zeros(3, 2, 64, dtype=BF16), value=torch.zeros(3, 2, 64, dtype=BF16), key_cache=torch.zeros(5, 16, 2, 64, dtype=BF16),
                value_cache=torch.zeros(5, 16, 2, 64, dtype=BF16), slots=torch.zeros(3, dtype=torch.long))
    call.update(changes)
    return call


@pytest.mark.parametrize("changes,says", [
    ({}, "cuda"),
    (dict(value=torch.zeros(3, 2, 32, dtype=BF16)), "value like key"),
    (dict(key_cache=torch.zeros(5, 16, 3, 64, dtype=BF16)), "key_cache to have shape"),
    (dict(key_cache=torch.zeros(5, 16, 2, 64, dtype=torch.float16)), "or torch.float8_e4m3fn"),
    (dict(value_cache=torch.zeros(4, 16, 2, 64, dtype=BF16)), "one shape"),
    (dict(value_cache=torch.zeros(5, 16, 64, 2, dtype=BF16).transpose(2, 3)), "unit stride"),
    (dict(key_cache=torch.zeros(5, 0, 2, 64, dtype=BF16)), "one place or more"),
    (dict(slots=torch.zeros(3)), "slots"),
    (dict(slots=torch.zeros(2, dtype=torch.long)), "slots"),
    (dict(positions=torch.zeros(3, dtype=torch.long)), "together"),
    (dict(query=torch.zeros(3, 4, 64, dtype=BF16)), "frequencies and positions with a query"),
    (dict(query_output=torch.zeros(3, 4, 64, dtype=BF16)), "with a query only"),
    (dict(query=torch.zeros(2, 4, 64, dtype=BF16), positions=torch.zeros(3, dtype=torch.long), frequencies=torch.ones(8)), "key's tokens"),
    (dict(key_scale=torch.ones(1)), "no key_scale"),
    (dict(key_cache=torch.zeros(5, 16, 2, 64).to(FP8), value_cache=torch.zeros(5, 16, 2, 64).to(FP8), value_scale=torch.ones(3)), "value_scale to be 1 or 2"),
    (dict(key=torch.zeros(3, 0, 64, dtype=BF16), value=torch.zeros(3, 0, 64, dtype=BF16)), "one key head")])
def test_append_refuses(changes, says):
    with pytest.raises(AssertionError, match=says):
        append_kv(**_append_call(**changes))


def _attention_call(**changes):
    call = dict(query=torch.zeros(4, 4, 64, dtype=BF16), key_cache=torch.zeros(5, 16, 2, 64, dtype=BF16), value_cache=torch.zeros(5, 16, 2, 64, dtype=BF16),
                page_table=torch.zeros(2, 3, dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32))
    call.update(changes)
    return call


def _caches(*shape, dtype=BF16):
    return dict(key_cache=torch.zeros(*shape).to(dtype), value_cache=torch.zeros(*shape).to(dtype))


@pytest.mark.parametrize("changes,says", [
    ({}, "cuda"),
    (dict(query=torch.zeros(4, 4, 64)), "bfloat16 or torch.float16"),
    (dict(query=torch.zeros(4, 3, 64, dtype=BF16)), "multiple of kv_heads"),
    (dict(query=torch.zeros(3, 4, 64, dtype=BF16)), "Expected starts"),
    (dict(query=torch.zeros(4, 4, 8, dtype=BF16), **_caches(5, 16, 2, 8)), "from 16 to 256"),
    (dict(query=torch.zeros(4, 4, 72, dtype=BF16), **_caches(5, 16, 2, 72, dtype=FP8)), "multiple of 16"),
    (dict(query=torch.zeros(4, 4, 136, dtype=BF16), **_caches(5, 16, 2, 136)), "multiple of 16"),
    (dict(query=torch.zeros(4, 4, 272, dtype=BF16), **_caches(5, 16, 2, 272)), "from 16 to 256"),
    (_caches(5, 12, 2, 64), "multiple of 8"),
    (_caches(0, 16, 2, 64), "a page"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.long)), "page_table"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()), "unit stride"),
    (dict(page_table=torch.zeros(1, dtype=torch.int32).expand(2, (1 << 23) + 1)), "unit stride|2\\^27"),
    (dict(lengths=torch.ones(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.ones(2, dtype=torch.long)), "lengths"),
    (dict(starts=torch.ones(2, dtype=torch.int32)), "starts"),
    (dict(mask=torch.ones(3, 2, dtype=torch.bool)), "mask"),
    (dict(mask=torch.ones(4, 2)), "mask"),
    (dict(scale=0.0), "scale"),
    (dict(scale=math.nan), "scale"),
    (dict(key_scale=torch.ones(1)), "no key_scale"),
    (dict(out_scale=torch.ones(2)), "out_scale"),
    (dict(output=torch.zeros(4, 4, 64)), "output"),
    (dict(out_scale=torch.ones(1), output=torch.zeros(4, 4, 64, dtype=BF16)), "output")])
def test_attention_refuses(changes, says):
    with pytest.raises(AssertionError, match=says):
        tree_attention(**_attention_call(**changes))


def test_operators_have_no_cpu_path():
    for op, call in ((torch.ops._HFRK_C.rotary, lambda: (torch.zeros(1, 1, 16, dtype=BF16), torch.zeros(1, dtype=torch.long), torch.ones(8), 1.0, False,
                                                         torch.zeros(1, 1, 16, dtype=BF16))),):
        with pytest.raises((NotImplementedError, RuntimeError)):
            op(*call())


# ---- the C ABI ----------------------------------------------------------------------------------------------------------

def _append_args(**changes):
    a = _capi.AppendArgs()
    for name in ("query", "query_output", "key", "value", "key_cache", "value_cache", "slots", "positions", "frequencies"):
        setattr(a, name, 4096)
    for name, v in {**dict(tokens=1, heads=2, kv_heads=1, head_dim=64, rotated=64, pages=1, page_size=16, dtype=_capi.BF16,
                           cache_dtype=_capi.BF16, magnitude=1.0), **changes}.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("changes,status", [
    (dict(tokens=-1), _capi.BAD_SHAPE), (dict(head_dim=0), _capi.BAD_SHAPE), (dict(head_dim=1025), _capi.BAD_SHAPE), (dict(rotated=63), _capi.BAD_SHAPE),
    (dict(rotated=66), _capi.BAD_SHAPE), (dict(rotated=-2), _capi.BAD_SHAPE), (dict(positions=None), _capi.BAD_SHAPE), (dict(slots=None), _capi.BAD_SHAPE),
    (dict(query=None), _capi.BAD_SHAPE), (dict(value_cache=None), _capi.BAD_SHAPE), (dict(page_size=0), _capi.BAD_SHAPE), (dict(pages=-1), _capi.BAD_SHAPE),
    (dict(dtype=_capi.FP8_E4M3FN), _capi.BAD_DTYPE), (dict(cache_dtype=_capi.F16), _capi.BAD_DTYPE), (dict(key_scale=4096), _capi.BAD_DTYPE),
    (dict(heads=70000), _capi.BAD_SHAPE), (dict(tokens=0), _capi.SUCCESS), (dict(heads=0, kv_heads=0), _capi.SUCCESS)])
def test_append_status(changes, status):
    a = _append_args(**changes)
    assert _capi.load().hfrk_append_kv(ctypes.byref(a), None) == status


def _attention_args(**changes):
    a = _capi.AttentionArgs()
    for name in ("query", "output", "key_cache", "value_cache", "page_table", "lengths"):
        setattr(a, name, 4096)
    for name in ("query_token_stride", "query_head_stride", "output_token_stride", "output_head_stride", "key_page_stride", "key_place_stride",
                 "key_cache_head_stride", "value_page_stride", "value_place_stride", "value_cache_head_stride"):
        setattr(a, name, 64)
    for name, v in {**dict(tokens=2, seqs=2, heads=4, kv_heads=2, head_dim=64, pages=3, page_size=16, table_columns=300, dtype=_capi.BF16,
                           cache_dtype=_capi.BF16, scale=0.125), **changes}.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("changes,status", [
    (dict(heads=3), _capi.BAD_SHAPE), (dict(head_dim=8), _capi.BAD_SHAPE), (dict(head_dim=68), _capi.BAD_SHAPE), (dict(head_dim=136), _capi.BAD_SHAPE),
    (dict(head_dim=264), _capi.BAD_SHAPE), (dict(head_dim=72, cache_dtype=_capi.FP8_E4M3FN), _capi.BAD_SHAPE), (dict(page_size=4), _capi.BAD_SHAPE),
    (dict(page_size=20), _capi.BAD_SHAPE), (dict(pages=0), _capi.BAD_SHAPE), (dict(table_columns=0), _capi.BAD_SHAPE),
    (dict(table_columns=(1 << 23) + 1), _capi.BAD_SHAPE), (dict(tokens=3), _capi.BAD_SHAPE), (dict(seqs=0), _capi.BAD_SHAPE), (dict(scale=0.0), _capi.BAD_SHAPE),
    (dict(scale=math.nan), _capi.BAD_SHAPE), (dict(tokens=1 << 27, seqs=1 << 20), _capi.BAD_SHAPE), (dict(query=None), _capi.BAD_SHAPE),
    (dict(lengths=None), _capi.BAD_SHAPE), (dict(query=4104), _capi.BAD_ALIGNMENT), (dict(key_cache=4104), _capi.BAD_ALIGNMENT),
    (dict(output=4104), _capi.BAD_ALIGNMENT), (dict(query_head_stride=68), _capi.BAD_ALIGNMENT), (dict(value_place_stride=66), _capi.BAD_ALIGNMENT),
    (dict(cache_dtype=_capi.FP8_E4M3FN, key_page_stride=72), _capi.BAD_ALIGNMENT), (dict(cache_dtype=_capi.F16), _capi.BAD_DTYPE),
    (dict(dtype=_capi.FP8_E4M3FN), _capi.BAD_DTYPE), (dict(value_scale=4096), _capi.BAD_DTYPE), (dict(tokens=0), _capi.SUCCESS),
    (dict(), _capi.BAD_ALIGNMENT)])  # the last: no workspace, where one is needed
def test_attention_status(changes, status):
    a = _attention_args(**changes)
    assert _capi.load().hfrk_tree_attention(ctypes.byref(a), None, 0, None) == status


def test_attention_workspace():
    lib = _capi.load()
    a = _attention_args()
    need = lib.hfrk_tree_attention_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.hfrk_tree_attention(ctypes.byref(a), 4096, need - 1, None) == _capi.EXCEEDS_SCRATCH
    assert lib.hfrk_tree_attention(ctypes.byref(a), 4100, need, None) == _capi.BAD_ALIGNMENT
    assert lib.hfrk_tree_attention_workspace_bytes(ctypes.byref(_attention_args(table_columns=8))) == 0   # 128 tokens at most: never split
    assert lib.hfrk_tree_attention_workspace_bytes(ctypes.byref(_attention_args(tokens=0))) == 0
    assert lib.hfrk_tree_attention_workspace_bytes(ctypes.byref(_attention_args(heads=3))) == 0
    # it is bounded by the work that the card can have at once, not by the lengths
    assert lib.hfrk_tree_attention_workspace_bytes(ctypes.byref(_attention_args(table_columns=1 << 23, head_dim=256, tokens=64))) < 300 << 20


# ---- tracing ------------------------------------------------------------------------------------------------------------

def test_wrappers_under_fake_tensors():
    with FakeTensorMode():
        def empty(*shape, dtype=BF16):
            return torch.empty(*shape, device="cuda", dtype=dtype)
        query, rows = empty(6, 8, 64), empty(6, 2, 64)
        cache = empty(10, 16, 2, 64, dtype=FP8)
        positions, frequencies = empty(6, dtype=torch.long), empty(32, dtype=torch.float64)
        assert rotary(query, positions, frequencies).shape == query.shape
        assert append_kv(rows, rows, cache, empty(10, 16, 2, 64, dtype=FP8), positions, positions, frequencies, query=query).shape == query.shape
        assert append_kv(rows, rows, cache, empty(10, 16, 2, 64, dtype=FP8), positions) is None
        args = cache, cache, empty(2, 5, dtype=torch.int32), empty(2, dtype=torch.int32)
        out = tree_attention(query, *args)
        assert out.shape == query.shape and out.dtype == BF16
        assert tree_attention(query, *args, out_scale=empty(1, dtype=torch.float32)).dtype == FP8


@pytest.mark.parametrize("tokens", [6, 0, 700])
def test_the_attention_block_under_fake_tensors(tokens):
    from hf_rocm_kernels.combined_ops.llama_attention import llama_attention_combined_ops
    with FakeTensorMode():
        def empty(*shape, dtype=BF16):
            return torch.empty(*shape, device="cuda", dtype=dtype)
        scale = empty(1, dtype=torch.float32)
        hidden, residual = empty(tokens, 512), empty(tokens, 512)
        out, residual_out = llama_attention_combined_ops(
            hidden, residual, empty(512), 1e-5, empty(768, 512, dtype=FP8), empty(768, dtype=torch.float32), scale, empty(512, 512, dtype=FP8), scale,
            scale, empty(10, 16, 2, 64, dtype=FP8), empty(10, 16, 2, 64, dtype=FP8), empty(tokens, dtype=torch.int32), empty(tokens, dtype=torch.long),
            empty(32, dtype=torch.float64), empty(2, 5, dtype=torch.int32), empty(2, dtype=torch.int32), empty(3, dtype=torch.int32),
            empty(tokens, 9, dtype=torch.bool), key_scale=scale, value_scale=scale)
        assert out.shape == hidden.shape and out.dtype == BF16 and residual_out is residual


# ---- frequencies and the Torch forms --------------------------------------------------------------------------------------

def test_frequencies():
    f, magnitude = rotary_frequencies(64, 10000.0, device="cpu")
    assert magnitude == 1.0 and f.dtype == torch.float64 and f.shape == (32,)
    assert all(abs(float(f[j]) - 10000.0 ** (-2 * j / 64)) <= 1e-15 for j in range(32))
    halved, _ = rotary_frequencies(64, 10000.0, {"rope_type": "linear", "factor": 2.0}, device="cpu")
    assert torch.equal(halved, f / 2)
    # kept above 4 turns within 1024 positions, divided by 8 below one, between them by the turns
    by_turns, _ = rotary_frequencies(64, 10000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                                   "original_max_position_embeddings": 1024}, device="cpu")
    for j in range(32):
        turns = 1024 * float(f[j]) / (2 * math.pi)
        kept = 1.0 if turns > 4 else 0.0 if turns < 1 else (turns - 1) / 3
        assert math.isclose(float(by_turns[j]), float(f[j]) * (kept + (1 - kept) / 8), rel_tol=1e-14)
    yarn, magnitude = rotary_frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}, device="cpu")
    assert math.isclose(magnitude, 0.1 * math.log(4.0) + 1.0)
    first, last = (64 * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(10000.0)) for n in (32, 1))
    for j in range(32):
        divided = min(max((j - math.floor(first)) / (math.ceil(last) - math.floor(first)), 0.0), 1.0)
        assert math.isclose(float(yarn[j]), float(f[j]) * (1 - divided + divided / 4), rel_tol=1e-14)
    assert rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64, "attention_factor": 0.5}, device="cpu")[1] == 0.5
    with pytest.raises(ValueError, match="rope_type"):
        rotary_frequencies(64, scaling={"rope_type": "dynamic", "factor": 2.0}, device="cpu")
    with pytest.raises(AssertionError):
        rotary_frequencies(63, device="cpu")


@pytest.mark.parametrize("interleaved", [False, True])
def test_torch_forms_agree_with_the_oracle(interleaved):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 4, 64, generator=g).double()
    positions = torch.randint(0, 1 << 20, (5,), generator=g)
    f = rotary_frequencies(48, device="cpu")[0]
    want = oracle.rotary(x, positions, f, interleaved, 0.9)[0]
    assert (reference_rotary(x, positions, f, interleaved, 0.9) - want).abs().max() < 1e-9
    key, value = (torch.randn(5, 2, 64, generator=g).to(torch.float16) for _ in range(2))
    caches = [torch.zeros(3, 16, 2, 64, dtype=torch.float16) for _ in range(2)]
    slots = torch.tensor([0, 47, -1, 48, 17])
    reference_append_kv(key, value, *caches, slots, positions, f, interleaved)
    turned = oracle.rotary(key, positions, f, interleaved)[0].to(torch.float16)
    assert torch.equal(caches[1][2, 15], value[1]) and torch.equal(caches[0][1, 1], turned[4]) and int((caches[1] != 0).any(-1).any(-1).sum()) == 3
    query = torch.randn(7, 4, 64, generator=g).to(torch.float16)
    table, lengths, starts = torch.tensor([[2, 0], [1, -1]], dtype=torch.int32), torch.tensor([20, 16]), torch.tensor([0, 3, 7])
    caches = [torch.randn(3, 16, 2, 64, generator=g).to(torch.float16) for _ in range(2)]
    caches[1][1, 14, 1, 5] = math.nan
    mask = torch.rand(7, 4, generator=g) < 0.5
    for m in (None, mask):
        want = oracle.attention(query, *caches, table, lengths, starts, m, 0.125)[0]
        got = reference_tree_attention(query, *caches, table, lengths, starts, m, 0.125)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and (got - want)[~torch.isnan(want)].abs().max() < 1e-12


def test_package_lists_its_operators():
    for name in ("rotary", "rotary_frequencies", "append_kv", "tree_attention"):
        assert name in hf_rocm_kernels.__all__ and callable(getattr(hf_rocm_kernels, name))


def test_whole_call_operators_take_no_meta_tensor_among_others():
    """One meta tensor among tensors with data: no result that nobody computed; on meta tensors alone, shapes."""
    ops = torch.ops._HFRK_C

    def tensors(device, other=None, at=None):
        def make(i, *shape, dtype=BF16):
            return torch.empty(*shape, dtype=dtype, device=other if i == at else device)
        return (make(0, 4, 4, 64), make(1, 4, 2, 64), make(2, 5, 16, 2, 64), make(3, 4, dtype=torch.long), make(4, 32, dtype=torch.float64),
                make(5, 2, 3, dtype=torch.int32), make(6, 2, dtype=torch.int32))

    turn = lambda q, k, c, p, f, table, n: ops.rotary_new(q, p, f, 1.0, False)
    append = lambda q, k, c, p, f, table, n: ops.append_kv_new(k, k, c, c, p, p, f, 1.0, False, q, None, None)
    attend = lambda q, k, c, p, f, table, n: ops.tree_attention_new(q, c, c, table, n, None, None, None, None, None, None)
    alone = tensors("meta")
    assert turn(*alone).shape == (4, 4, 64) and append(*alone)[0] and append(*alone)[1].shape == (4, 4, 64) and attend(*alone).shape == (4, 4, 64)
    for at, call in ((3, turn), (4, turn), (2, attend), (5, attend), (6, attend)):
        assert call(*tensors("cpu", "meta", at)) is None
    for at in (1, 2, 3, 4):
        assert append(*tensors("cpu", "meta", at)) == (False, None)


YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("changes,magnitude", [
    (dict(mscale=1.0, mscale_all_dim=1.0), 1.0), (dict(mscale=0.707, mscale_all_dim=0.707), 1.0),
    (dict(mscale=1.0, mscale_all_dim=0.5), (0.1 * math.log(40.0) + 1.0) / (0.05 * math.log(40.0) + 1.0)),
    (dict(mscale=1.0, mscale_all_dim=0.5, factor=0.5), 1.0), (dict(mscale=1.0, mscale_all_dim=0.5, attention_factor=0.25), 0.25),
    (dict(mscale=1.0), 0.1 * math.log(40.0) + 1.0), (dict(mscale=None, mscale_all_dim=None, truncate=None), 0.1 * math.log(40.0) + 1.0),
    (dict(mscale=0.0, mscale_all_dim=0), 0.1 * math.log(40.0) + 1.0)])
def test_magnitude_of_yarn_entries(changes, magnitude):
    assert math.isclose(rotary_frequencies(64, scaling={**YARN, **changes}, device="cpu")[1], magnitude, rel_tol=1e-15)


def test_a_yarn_ramp_between_whole_pairs():
    """truncate false: the ramp's ends are not rounded outwards."""
    plain = rotary_frequencies(64, device="cpu")[0]
    got = rotary_frequencies(64, scaling={**YARN, "truncate": False, "beta_fast": 16, "beta_slow": 2}, device="cpu")[0]
    first, last = (64 * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(10000.0)) for n in (16, 2))
    for j in range(32):
        divided = min(max((j - first) / (last - first), 0.0), 1.0)
        assert math.isclose(float(got[j]), float(plain[j]) * (1 - divided + divided / 40), rel_tol=1e-13)
    assert not torch.equal(got, rotary_frequencies(64, scaling={**YARN, "beta_fast": 16, "beta_slow": 2}, device="cpu")[0])


@pytest.mark.parametrize("scaling,says", [
    ({**YARN, "mscale": 0.7}, "mscale_all_dim"), ({**YARN, "mscale_all_dim": 1.0}, "mscale_all_dim"), ({**YARN, "long_factor": [1.0]}, "long_factor"),
    ({"rope_type": "linear", "factor": 2.0, "attention_factor": 1.5}, "attention_factor"), ({"type": "default", "mrope_section": [16, 24, 24]}, "mrope_section"),
    ({"rope_type": "default", "factor": 4.0}, "factor"), ({**YARN, "rope_theta": 500000.0}, "rope_theta"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 1024, "truncate": False}, "truncate")])
def test_entries_that_are_not_understood_are_refused(scaling, says):
    with pytest.raises(ValueError, match=says):
        rotary_frequencies(64, scaling=scaling, device="cpu")


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default", "rope_theta": 10000.0}, {"type": "default", "factor": 1.0, "original_max_position_embeddings": 2048, "finetuned": True},
    {"rope_type": "linear", "factor": 1.0, "attention_factor": None, "partial_rotary_factor": 0.5}])
def test_entries_with_keys_that_change_nothing(scaling):
    assert torch.equal(rotary_frequencies(64, scaling=scaling, device="cpu")[0], rotary_frequencies(64, device="cpu")[0])


@pytest.mark.parametrize("tokens,seqs,kv_heads,status", [
    (1 << 16, 1 << 16, 8, _capi.BAD_ALIGNMENT), (1 << 18, 1 << 18, 2, _capi.BAD_SHAPE), (1 << 17, 1 << 17, 8, _capi.BAD_SHAPE),
    (1 << 20, 1 << 20, 1, _capi.BAD_SHAPE), (1 << 15, 1 << 14, 64, _capi.BAD_ALIGNMENT), (1 << 16, 1 << 16, 64, _capi.BAD_SHAPE)])
def test_batches_whose_list_of_work_would_take_seconds_are_refused(tokens, seqs, kv_heads, status):
    """Every workgroup makes the list: workgroups times sequences are bounded.  (Those that are taken lack a workspace here.)"""
    a = _attention_args(tokens=tokens, seqs=seqs, heads=kv_heads, kv_heads=kv_heads)
    assert _capi.load().hfrk_tree_attention(ctypes.byref(a), None, 0, None) == status


@pytest.mark.parametrize("seqs,kv_heads,status", [(1024, 8192, _capi.BAD_ALIGNMENT), (2048, 8192, _capi.BAD_SHAPE)])
def test_launches_of_more_threads_than_32_bits_count_are_refused(seqs, kv_heads, status):
    """A launch of 2^24 + n workgroups of 256 threads runs n of them, without an error."""
    a = _attention_args(tokens=seqs, seqs=seqs, heads=kv_heads, kv_heads=kv_heads)
    assert _capi.load().hfrk_tree_attention(ctypes.byref(a), None, 0, None) == status
