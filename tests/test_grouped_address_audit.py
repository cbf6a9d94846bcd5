"""Address audit of the products grouped by expert on the host, no GPU: which tile a workgroup finds, and every address that csrc/grouped_gemm.hip and the grouped
form of csrc/tiled_gemm_kernel.h make of the rows that a tile picks, restated from the source and checked against what it points into (rules as in
test_address_audit.py: a live access lies inside its buffer, a suppressed one at or beyond its end without wrapping round)."""
import os
import random
import re

import numpy as np
import pytest

from hf_rocm_kernels import _capi
from test_address_audit import U32

KB, XCDS, OUTSIDE, MOST = 128, 8, 0x7FFFFFF0, 1 << 21
CSRC = os.path.join(os.path.dirname(_capi.LIB_PATH), os.pardir, "csrc")
LANE = np.arange(64)


def _shapes():
    """(TM, TN, WM, WN, stages or halves in LDS, halves, waves that only load) of the kernels built for groups."""
    with open(os.path.join(CSRC, "grouped_gemm.h")) as f:
        lists = re.findall(r"#define HFRK_GROUP_(SHAPES|PAIRED)\(X\)((?:.*\\\n)*.*)", f.read())
    shapes = []
    for name, rows in lists:
        for row in re.findall(r"X\((\d), (\d), (\d), (\d), (\d), (\d), \d\)", rows):
            index, TM, TN, WM, WN, NST = map(int, row)
            assert index == len(shapes)
            halves = name == "PAIRED" or TM * WM * WN >= 32
            shapes.append((TM, TN, WM, WN, NST, halves, 4 if name == "SHAPES" and TM < 4 else 0))
    assert len(shapes) == 5
    return shapes


SHAPES = _shapes()


def _bound(count, experts, bm):
    return count // bm + min(experts, count)


def _find(block, offsets, count, bm, tiles_n):
    """find_tile: (expert, first row, rows, tile, rows of tiles) of a workgroup, or None."""
    edge = np.clip(np.asarray(offsets, dtype=np.int64), 0, count)
    tiles = np.where(edge[1:] > edge[:-1], -(-(edge[1:] - edge[:-1]) // bm), 0)
    upto = np.cumsum(tiles)
    total = int(upto[-1]) * tiles_n
    x, slot, per, extra = block % XCDS, block // XCDS, total // XCDS, total % XCDS
    if slot >= per + (x < extra):
        return None
    id = x * per + min(x, extra) + slot
    e = int(np.argmax(upto * tiles_n > id))
    left = id - int(upto[e] - tiles[e]) * tiles_n
    assert 0 <= left < tiles[e] * tiles_n
    return e, int(edge[e]), int(edge[e + 1] - edge[e]), left, int(tiles[e])


@pytest.mark.parametrize("bm", [16, 128, 256])
@pytest.mark.parametrize("seed", range(6))
def test_every_tile_of_every_group_is_found_once(bm, seed):
    rng = random.Random(seed)
    experts, count, tiles_n = rng.choice((1, 7, 64, 65, 128, 200, 512)), rng.choice((1, 5, 100, 900)), rng.randint(1, 5)
    offsets = sorted(rng.randint(0, count) for _ in range(experts + 1))
    if seed % 2:
        offsets[0], offsets[-1] = 0, count
    grid = _bound(count, experts, bm) * tiles_n
    found = [t for t in (_find(b, offsets, count, bm, tiles_n) for b in range(grid)) if t]
    wanted = {(e, i) for e in range(experts) for i in range(-(-(offsets[e + 1] - offsets[e]) // bm) * tiles_n)}
    assert len(found) == len(wanted) and {(t[0], t[3]) for t in found} == wanted
    assert all(t[1] == offsets[t[0]] and t[2] == offsets[t[0] + 1] - offsets[t[0]] for t in found)


@pytest.mark.parametrize("offsets", [[5, 3, 900, -7], [0, 40, 0, 40], [-(1 << 31), (1 << 31) - 1, 0, 12], [99, 98, 97, 96]])
def test_offsets_that_are_none_lead_to_rows_that_are_there(offsets):
    for bm in (16, 128):
        for block in range(_bound(40, 3, bm) * 3):
            t = _find(block, offsets, 40, bm, 3)
            assert t is None or (0 <= t[1] and t[2] > 0 and t[1] + t[2] <= 40 and t[3] < t[4] * 3)


def _loads(rows, halves, NL, loader):
    """Rows that the loads of a wave fetch, whatever its number among those that load is."""
    q = np.arange(rows * KB // (1024 * NL))[:, None]
    return ((q >> 1) * NL + loader) * 16 + (LANE >> 2) if halves else (q * NL + loader) * 8 + (LANE >> 3)


@pytest.mark.parametrize("shape", range(5))
@pytest.mark.parametrize("k,a_rows", [(16, 1), (2064, 700), (MOST, 1020), (4096, (1 << 19) - 1200)])
def test_rows_that_a_tile_picks(shape, k, a_rows):
    TM, TN, WM, WN, NST, halves, LW = SHAPES[shape]
    NW, BM = WM * WN, 32 * TM * WM
    NL = LW or NW
    assert a_rows * k <= OUTSIDE - MOST
    numbers = np.array([0, a_rows - 1, -1, a_rows, (1 << 31) - 1, -(1 << 31)])
    for rows_a in {1, BM // 2 + 1, BM}:
        seen = []
        for wave in range(NW + LW):
            loader = wave - (NW if LW else 0)
            row = _loads(BM, halves, NL, loader)
            offset = (row * 4) % U32                       # of its number, in a buffer over the tile's own
            inside = offset + 4 <= rows_a * 4
            # a wave that only multiplies has a number below zero, and so have some of its rows: it asks for none, and the buffer would give none of those
            assert (inside == ((row >= 0) & (row < rows_a))).all()
            if loader < 0:
                assert (row < 0).any()
                continue
            seen += row[inside].tolist()
            for number in numbers:
                there = inside & (0 <= number < a_rows)
                for at in {0, k // KB // 2, (k - 1) // KB}:
                    for piece in range(0, KB, 16):
                        if at * KB + piece >= k:
                            continue
                        offset = np.where(there, number * k + piece, OUTSIDE)
                        records = a_rows * k - at * KB
                        live = offset + 16 <= records
                        assert (offset >= 0).all() and (live == there).all()
        assert set(seen) == set(range(rows_a))
        # the scales: of one row each, or one for all
        for stride in (0, 1):
            for number in numbers:
                there = 0 <= number < a_rows
                offset = number * stride * 4 if there else OUTSIDE
                assert (offset + 4 <= ((a_rows - 1) * stride + 1) * 4) == there


@pytest.mark.parametrize("shape", range(5))
def test_waves_lds_and_loads_in_flight(shape):
    TM, TN, WM, WN, NST, halves, LW = SHAPES[shape]
    NW, BM, BN, NL = WM * WN, 32 * TM * WM, 32 * TN * WN, LW or WM * WN
    ring = (BM + BN) * (KB // 2 if halves else KB) * NST
    assert ring <= 160 * 1024 and NW * 32 * (TN * 32 + 4) * 4 <= ring and (NW + LW) * 64 <= 1024
    loads = 0
    for rows in (BM, BN):
        per_wave = rows * KB // (1024 * NL)
        assert per_wave * 1024 * NL == rows * KB and (not halves or per_wave % 2 == 0)
        loads += per_wave
        fetched = np.concatenate([_loads(rows, halves, NL, w) for w in range(NL)])
        assert (np.bincount(fetched.ravel(), minlength=rows) == 8).all()  # each of a row's eight pieces
    assert (NST // 2 - 1 if halves else NST - 1) * loads <= 63


@pytest.mark.parametrize("k", [16, 112, 128, 144, 1040, MOST])
def test_the_rows_kernel_asks_for_nothing_behind_a_row(k):
    """Pieces of 16 bytes, two of each 128-byte chunk a lane: those at or behind k are asked for outside the buffer, whichever chunk is prefetched."""
    for KW in (4, 8):
        chunks = -(-k // KB)
        last = (chunks - 1 + 3 * KW) * KB + 64 + 48
        assert OUTSIDE + last < U32 and (127 * MOST + k) < 1 << 31
        for c in {0, chunks // 2, chunks - 1, chunks, chunks - 1 + 3 * KW}:
            by = c * KB + np.array([0, 64])[:, None] + (LANE >> 4) * 16
            live = by < k
            assert (by[live] + 16 <= k).all() and (OUTSIDE + by[~live] >= (1 << 31) - MOST).all()
