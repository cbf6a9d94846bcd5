"""The attention's list of work on the host, no GPU: what csrc/tree_attention.h's find_part deals out, restated from the source, against the grid and the
workspace that csrc/tree_attention.hip bounds from the sizes alone; the workspace's bytes are the library's own answer."""
import ctypes
import random

import numpy as np
import pytest

from hf_rocm_kernels import _capi

F = np.float32
CUS = 256


def ceil_div(a, b):
    return -(-a // b)


def splits_of(tiles, chunk, ulp=0):
    """ceil(tiles / chunk) by the device's reciprocal, which may be off by a step either way."""
    r = F(1) / F(chunk)
    if ulp:
        r = np.nextafter(r, F(2) if ulp > 0 else F(0))
    return max(1, int(F(F(tiles + chunk) - F(0.5)) * r))


@pytest.mark.parametrize("ulp", [-1, 0, 1])
def test_quotients(ulp):
    for tiles in [*range(0, 4000, 7), (1 << 20) - 1, 1 << 20]:
        for chunk in (1, 2, 3, 5, 7, 11, 100, 999, 4096, (1 << 20) - 1):
            assert splits_of(tiles, chunk, ulp) == max(1, ceil_div(tiles, chunk))


def decompose(tokens, seqs, group, kv_heads, head_dim, places):
    """(rows of a block, workgroups at once, shares, grid / kv_heads, slots)"""
    per = ceil_div(tokens, seqs) * group
    tiles = ceil_div(places, 128)
    few = (tokens * group // 32 + seqs) * tiles * kv_heads
    shared = per > 32 and few > (4 if head_dim > 128 else 24) * CUS
    rows = 16 if per <= 16 else 32 if per <= 32 or not shared else 128 if per <= 128 or head_dim > 128 else 256
    work = CUS if rows == 256 or head_dim > 128 else 2 * CUS
    shares = 2 if seqs > 1 else 1
    blocks, most = tokens * group // rows + seqs, shares * max(1, work // kv_heads)
    items = min(most + blocks, blocks * tiles)
    return rows, work, shares, items, min(2 * most, blocks * tiles) if tiles > 1 else 0


def dealt_out(blocks, tiles, room, shares):
    """The chunk that find_part takes, as there in 32-bit floats."""
    total, least = sum(b * t for b, t in zip(blocks, tiles)), sum(blocks)
    items_of = lambda chunk: sum(b * splits_of(t, chunk) for b, t in zip(blocks, tiles))
    chunk = share = max(1, ceil_div(total, room))
    if shares > 1 and least > 0:
        best, at_once = F(3e38), 0
        for k in range(1, shares + 2):
            now = ceil_div(share, k) if k <= shares else share * at_once // room + 1
            if k > shares and (at_once <= room or least > room):
                break
            items = items_of(now)
            if k == 1:
                at_once = items
            ends = F(now) if items <= room else F((F(total) + F(2) * F(items)) / F(room) + F(0.5) * F(now))
            if ends < best:
                best, chunk = ends, now
    return chunk


def library_bytes(tokens, seqs, group, kv_heads, head_dim, page_size, columns):
    a = _capi.AttentionArgs()
    for name in ("query", "output", "key_cache", "value_cache", "page_table", "lengths", "starts"):
        setattr(a, name, 1 << 20)
    a.tokens, a.seqs, a.heads, a.kv_heads, a.head_dim, a.pages = tokens, seqs, group * kv_heads, kv_heads, head_dim, 1
    a.page_size, a.table_columns, a.scale, a.dtype, a.cache_dtype = page_size, columns, 1.0, 1, 1  # bfloat16
    for name in ("query", "output"):
        setattr(a, name + "_token_stride", a.heads * head_dim)
        setattr(a, name + "_head_stride", head_dim)
    for name in ("key", "value"):
        setattr(a, name + "_page_stride", page_size * kv_heads * head_dim)
        setattr(a, name + "_place_stride", kv_heads * head_dim)
        setattr(a, name + "_cache_head_stride", head_dim)
    return _capi.load().hfrk_tree_attention_workspace_bytes(ctypes.byref(a))


def test_grid_and_workspace_hold_every_list():
    rng = random.Random(0)
    seen = set()
    for _ in range(6000):
        seqs, kv_heads, group = rng.choice([1, 2, 3, 5, 64, 65, 130]), rng.choice([1, 2, 3, 5, 8, 16, 100, 700]), rng.choice([1, 2, 4, 7, 16])
        head_dim, page_size = rng.choice([64, 128, 256]), rng.choice([8, 16, 64])
        counts = [rng.choice([0, 1, 1, 3, rng.randint(0, 200)]) for _ in range(seqs)]
        tokens = sum(counts) + rng.choice([0, 0, 5])
        if tokens == 0:
            continue
        columns = rng.choice([16, 200, 5000, 100000]) // page_size + 1
        places = columns * page_size
        lengths = [min(places, int(places * rng.random() ** rng.choice([1, 4]))) for _ in range(seqs)]
        rows, work, shares, items, slots = decompose(tokens, seqs, group, kv_heads, head_dim, places)
        partial, info, statistics = slots * kv_heads * rows * head_dim * 4, tokens * group * 16 if slots else 0, slots * kv_heads * rows * 8
        assert library_bytes(tokens, seqs, group, kv_heads, head_dim, page_size, columns) == partial + info + statistics
        blocks, tiles = [ceil_div(n * group, rows) for n in counts], [ceil_div(n, 128) for n in lengths]
        chunk = dealt_out(blocks, tiles, max(1, work // kv_heads), shares)
        splits = [splits_of(t, chunk) for t in tiles]
        assert sum(b * s for b, s in zip(blocks, splits)) <= items
        assert sum(b * s for b, s in zip(blocks, splits) if s > 1) <= slots
        for t, s in zip(tiles, splits):  # each tile is one split's
            even = ceil_div(t, s)
            parts = [(min(i * even, t), min((i + 1) * even, t)) for i in range(s)]
            assert parts[0][0] == 0 and parts[-1][1] == t and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        seen.add((rows, work, shares))
    assert len(seen) >= 9
