"""The router, the experts' sum, groups of few rows and the search for a group's tile from their own sources, on the CPU, lane by lane (lane_run.py), with every
tensor between pages that nothing may touch.  Test infrastructure only (see __init__.py)."""
import ctypes
import threading

import torch

from hf_rocm_kernels import _capi

from .lane_run import Memory, _run, build

_HEADERS = ("hfrk_internal.h", "skinny_gemm_args.h", "skinny_gemm_plan.h", "tiled_gemm.h", "grouped_gemm.h")
_SOURCES = ("grouped_gemm.hip", "experts.hip")
_TYPES = {torch.float16: _capi.F16, torch.bfloat16: _capi.BF16, torch.float32: _capi.FP32, torch.float8_e4m3fn: _capi.FP8_E4M3FN, torch.int8: _capi.INT8}
_lib = None
_loading = threading.Lock()


def _load():
    global _lib
    with _loading:
        if _lib is None:
            lib = ctypes.CDLL(build("groups", _HEADERS, _SOURCES, ("lanes.cpp", "groups.cpp")))
            for name in ("hfrk_route_experts", "hfrk_route_experts_workspace_bytes", "hfrk_combine_experts", "hfrk_grouped_gemm"):
                getattr(lib, name).restype, getattr(lib, name).argtypes = _capi.SIGNATURES[name]
            lib.lanes_tiles_bound.restype = ctypes.c_long
            _lib = lib
    return _lib


def _address(t):
    return None if t is None else t.data_ptr()


def _back(results, m):
    for t, at in results:
        ctypes.memmove(t.data_ptr(), at, t.numel() * t.element_size())


def route(logits, top, bias=None, scoring="softmax", renormalize=True, factor=1.0, mask=None, at_end=True, noise=0xff):
    """hfrk_route_experts of CPU tensors: (weights, experts, places, rows, offsets); results and workspace start as bytes of `noise`."""
    lib, m = _load(), Memory(at_end)
    tokens, experts = logits.shape
    out = [torch.empty((tokens, top)), *(torch.empty((tokens, top), dtype=torch.int32) for _ in range(2)), torch.empty(tokens * top, dtype=torch.int32),
           torch.empty(experts + 1, dtype=torch.int32)]
    at = [m.take(t.numel() * 4, noise) for t in out]
    need = lib.hfrk_route_experts_workspace_bytes(tokens, experts, top)
    workspace = m.take(need, noise) if need else None
    a = _capi.RouteArgs(logits=m.copy(logits), logits_stride=logits.stride(0), bias=m.copy(bias), mask=m.copy(mask), weights=at[0], experts=at[1], places=at[2], rows=at[3],
                        offsets=at[4], tokens=tokens, num_experts=experts, top=top, dtype=_TYPES[logits.dtype], sigmoid=int(scoring == "sigmoid"),
                        renormalize=int(renormalize), factor=factor)
    _run(lambda: lib.hfrk_route_experts(ctypes.byref(a), workspace, need, None))
    _back(zip(out, at), m)
    return tuple(out)


def combine(y, weights, places, base=None, at_end=True):
    """hfrk_combine_experts of CPU tensors."""
    lib, m = _load(), Memory(at_end)
    out = torch.empty((places.size(0), y.size(1)), dtype=y.dtype)
    at = m.take(out.numel() * 2, 0xff)
    pointers = [m.copy(t) for t in (y, weights, places, base)]
    _run(lambda: lib.hfrk_combine_experts(*pointers, at, *places.shape, y.size(1), y.size(0), _TYPES[y.dtype], None))
    _back([(out, at)], m)
    return out


def grouped(a, weight, scale_a, scale_b, offsets, rows, output, at_end=True):
    """hfrk_grouped_gemm of CPU tensors, ten rows a group in the mean at most; weight (experts, n, k) with unit stride along k.  Writes to output, which is returned."""
    lib, m = _load(), Memory(at_end)
    at = m.copy(output)
    experts, n, k = weight.shape
    args = _capi.GroupedArgs(a=m.copy(a), rows=m.copy(rows), b=m.copy(weight), expert_stride=weight.stride(0), output=at, scale_a=m.copy(scale_a), scale_b=m.copy(scale_b),
                             scale_b_expert_stride=0 if scale_b is None else scale_b.stride(0), offsets=m.copy(offsets), scale_a_stride=int(scale_a.numel() > 1),
                             scale_b_stride=int(scale_b is not None and scale_b.dim() == 2), b_stride=weight.stride(1), count=output.size(0), a_rows=a.size(0),
                             experts=experts, n=n, k=k, type=_TYPES[a.dtype], dtype=_TYPES[output.dtype])
    _run(lambda: lib.hfrk_grouped_gemm(ctypes.byref(args), None))
    _back([(output, at)], m)
    return output


def find_tiles(offsets, count, bm, tiles_n):
    """What each workgroup of the grid that the host bounds finds: (workgroups, 5), expert (-1: none), first row, rows, tile, rows of tiles; all lanes agree."""
    lib = _load()
    experts = offsets.numel() - 1
    grid = lib.lanes_tiles_bound(count, experts, bm) * tiles_n
    m = Memory(True)
    at, out = m.take(grid * 64 * 5 * 4), torch.empty((grid, 64, 5), dtype=torch.int32)
    given = m.copy(offsets)

    def call():
        lib.lanes_find_tiles(ctypes.c_void_p(given), experts, count, bm, tiles_n, grid, ctypes.c_void_p(at))
        return _capi.SUCCESS

    _run(call)
    _back([(out, at)], m)
    assert (out == out[:, :1]).all()
    return out[:, 0]
