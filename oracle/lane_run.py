"""The kernels of attention, rotation and append from their own sources, on the CPU, lane by lane (oracle/lanes), with every tensor between pages that
nothing may touch.  Test infrastructure only (see __init__.py).

The sources are taken as they are but for two things: statements of assembly (waits, and marks for the compiler) are left out, and the one array in a
launch's own LDS is a pointer.  A call runs in a child process, which an access outside the tensors, or lanes that meet at different places, end.  What it
cannot show: a missing wait or barrier, and an access that lands in another part of the same tensor or in its margin of up to 15 bytes."""
import ctypes
import faulthandler
import hashlib
import mmap
import os
import re
import shutil
import subprocess
import tempfile
import threading
from concurrent.futures import ThreadPoolExecutor

import torch

from hf_rocm_kernels import _capi

_HERE = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_HERE)
_CSRC = os.path.join(_ROOT, "hf-rocm-kernels_amd", "csrc")
_LANES = os.path.join(_HERE, "lanes")
_BUILD = os.path.join(_HERE, "_build")
_HEADERS = ("hfrk_internal.h", "overlap.h", "tree_attention.h", "tree_attention_kernel.h", "tree_attention_shared.h")
_SOURCES = ("rotary.hip", "tree_attention.hip", *(f"tree_attention_{kind}d{n}.hip" for kind in ("", "shared_") for n in (64, 128, 256)))
_PAGE = mmap.PAGESIZE
_MARGIN = 16 * _PAGE  # in front of a tensor and behind it
_lib = None
_loading = threading.Lock()


def _text(name):
    with open(os.path.join(_CSRC, name)) as f:
        text = f.read()
    text = re.sub(r"asm volatile\([^;]*;", ";", text)
    return re.sub(r"extern __shared__ float (\w+)\[\];", r"float* const \1 = reinterpret_cast<float*>(lanes::dynamic_memory);", text)


def build() -> str:
    """Compiles the sources, unless that has been done for these very ones; the library's path."""
    clang = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "clang++")
    texts = {name: _text(name) for name in _HEADERS + _SOURCES}
    with open(os.path.join(_LANES, "lanes.cpp")) as f:
        texts["lanes.cpp"] = f.read()
    digest = hashlib.sha256()
    for name in sorted(texts):
        digest.update(texts[name].encode())
    for path in (os.path.join(_LANES, "hip", "hip_runtime.h"), os.path.join(_ROOT, "include", "hfrk_gfx950.h")):
        with open(path, "rb") as f:
            digest.update(f.read())
    lib = os.path.join(_BUILD, f"lanes_{digest.hexdigest()[:16]}.so")
    if os.path.exists(lib):
        return lib
    os.makedirs(_BUILD, exist_ok=True)
    work = tempfile.mkdtemp(dir=_BUILD)
    try:
        for name, text in texts.items():
            with open(os.path.join(work, name), "w") as f:
                f.write(text)
        # (no floating-point contraction of a product and a sum that the source has apart; bytes of LDS are read as other types than written)
        flags = ["-x", "c++", "-std=c++17", "-O2", "-fPIC", "-w", "-fno-strict-aliasing", "-ffp-contract=off", "-D_Bool=bool", "-I" + _LANES, "-I" + work,
                 "-I" + os.path.join(_ROOT, "include")]
        def compiled(name):
            out = os.path.join(work, name + ".o")
            done = subprocess.run([clang, *flags, "-c", os.path.join(work, name), "-o", out], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
            assert done.returncode == 0, done.stdout
            return out
        with ThreadPoolExecutor(8) as pool:
            objects = list(pool.map(compiled, _SOURCES + ("lanes.cpp",)))
        subprocess.run([clang, "-shared", "-o", os.path.join(work, "all.so"), *objects], check=True)
        os.replace(os.path.join(work, "all.so"), lib)
    finally:
        shutil.rmtree(work)
    for name in os.listdir(_BUILD):  # of earlier sources
        if name.startswith("lanes_") and name.endswith(".so") and os.path.join(_BUILD, name) != lib:
            os.remove(os.path.join(_BUILD, name))
    return lib


def _load():
    global _lib
    with _loading:
        if _lib is None:
            lib = ctypes.CDLL(build())
            lib.hfrk_tree_attention_workspace_bytes.restype = ctypes.c_size_t
            _lib = lib
    return _lib


_libc = ctypes.CDLL(None)
_libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]


class Memory:
    """Tensors copied to memory of their own, flush with its end (or its beginning), between pages that may not be touched."""

    def __init__(self, at_end: bool):
        self.at_end, self.maps = at_end, []

    def take(self, nbytes: int, fill: int = 0) -> int:
        inside = max(-(-nbytes // _PAGE), 1) * _PAGE
        whole = mmap.mmap(-1, inside + 2 * _MARGIN, flags=mmap.MAP_SHARED | mmap.MAP_ANONYMOUS)  # (shared with the child that runs the call)
        base = ctypes.addressof(ctypes.c_char.from_buffer(whole))
        self.maps.append(whole)
        assert _libc.mprotect(base, _MARGIN, 0) == 0 and _libc.mprotect(base + _MARGIN + inside, _MARGIN, 0) == 0
        at = base + _MARGIN + ((inside - nbytes) // 16 * 16 if self.at_end else 0)  # (a multiple of 16, as allocations are)
        ctypes.memset(at, fill, nbytes)
        return at

    def copy(self, t):
        """The address of a copy of t, its strides and all that its storage holds kept."""
        if t is None:
            return None
        storage = t.untyped_storage()
        at = self.take(storage.nbytes())
        ctypes.memmove(at, storage.data_ptr(), storage.nbytes())
        return at + t.storage_offset() * t.element_size()


def _run(call) -> None:
    """call() in a child; its status must be that of success, and its end an ordinary one."""
    child = os.fork()
    if child == 0:
        status = 77
        faulthandler.disable()  # (the parent says what it means)
        try:
            status = call()
        finally:
            os._exit(status if 0 <= status < 77 else 77)
    ended = os.waitstatus_to_exitcode(os.waitpid(child, 0)[1])
    assert ended >= 0, f"signal {-ended}: 11 an access outside the tensors, 6 lanes that meet at different places"
    assert ended == _capi.SUCCESS, ended


def _dtype(t) -> int:
    return {torch.float16: _capi.F16, torch.bfloat16: _capi.BF16, torch.float8_e4m3fn: _capi.FP8_E4M3FN}[t.dtype]


def attention(query, key_cache, value_cache, page_table, lengths, starts=None, mask=None, scale=None, key_scale=None, value_scale=None, out_scale=None,
              output=None, at_end=True, noise=0xff):
    """hfrk_tree_attention of CPU tensors; the workspace starts as bytes of `noise`.  Writes to output, which is returned."""
    m = Memory(at_end)
    a = _capi.AttentionArgs()
    if output is None:
        output = torch.empty(query.shape, dtype=query.dtype if out_scale is None else torch.float8_e4m3fn)
    to = m.copy(output)
    mask = None if mask is None else mask.view(torch.uint8)
    for name, t in (("query", query), ("key_cache", key_cache), ("value_cache", value_cache), ("page_table", page_table), ("lengths", lengths), ("starts", starts),
                    ("mask", mask), ("key_scale", key_scale), ("value_scale", value_scale), ("out_scale", out_scale)):
        setattr(a, name, m.copy(t))
    a.output = to
    a.query_token_stride, a.query_head_stride = query.stride()[:2]
    a.output_token_stride, a.output_head_stride = output.stride()[:2]
    a.key_page_stride, a.key_place_stride, a.key_cache_head_stride = key_cache.stride()[:3]
    a.value_page_stride, a.value_place_stride, a.value_cache_head_stride = value_cache.stride()[:3]
    a.table_stride = page_table.stride(0)
    if mask is not None:
        a.mask_stride, a.mask_columns = mask.stride(0), mask.size(1)
    for name, t in (("key_scale_stride", key_scale), ("value_scale_stride", value_scale)):
        setattr(a, name, int(t is not None and t.numel() > 1))
    a.scale = query.size(2) ** -0.5 if scale is None else scale
    a.tokens, a.heads, a.head_dim = query.shape
    a.pages, a.page_size, a.kv_heads = key_cache.shape[:3]
    a.seqs, a.table_columns = page_table.shape
    a.dtype, a.cache_dtype = _dtype(query), _dtype(key_cache)
    lib = _load()
    nbytes = lib.hfrk_tree_attention_workspace_bytes(ctypes.byref(a))
    workspace = m.take(nbytes, noise)
    _run(lambda: lib.hfrk_tree_attention(ctypes.byref(a), ctypes.c_void_p(workspace), ctypes.c_size_t(nbytes), None))
    storage = output.untyped_storage()
    ctypes.memmove(storage.data_ptr(), to - output.storage_offset() * output.element_size(), storage.nbytes())
    return output


def _append_args(at, key, value, key_cache, value_cache, slots, positions, frequencies, interleaved, magnitude, query, query_output, key_scale, value_scale):
    """at: a tensor's address."""
    a = _capi.AppendArgs()
    for name, t in (("query", query), ("query_output", query_output), ("key", key), ("value", value), ("key_cache", key_cache), ("value_cache", value_cache),
                    ("slots", slots), ("positions", positions), ("frequencies", frequencies), ("key_scale", key_scale), ("value_scale", value_scale)):
        setattr(a, name, None if t is None else at(t))
    if query is not None:
        a.query_token_stride, a.query_head_stride = query.stride()[:2]
        a.output_token_stride, a.output_head_stride = query_output.stride()[:2]
        a.tokens, a.heads, a.head_dim = query.shape
        a.dtype = _dtype(query)
    if key is not None:
        a.key_token_stride, a.key_head_stride = key.stride()[:2]
        a.value_token_stride, a.value_head_stride = value.stride()[:2]
        a.key_page_stride, a.key_place_stride, a.key_cache_head_stride = key_cache.stride()[:3]
        a.value_page_stride, a.value_place_stride, a.value_cache_head_stride = value_cache.stride()[:3]
        a.tokens, a.kv_heads, a.head_dim = key.shape
        a.pages, a.page_size = key_cache.shape[:2]
        a.dtype, a.cache_dtype = _dtype(key), _dtype(key_cache)
        a.slots_wide = int(slots.dtype == torch.int64)
    if frequencies is not None:
        a.positions_wide, a.frequencies_wide = int(positions.dtype == torch.int64), int(frequencies.dtype == torch.float64)
        a.rotated, a.magnitude, a.interleaved = 2 * frequencies.numel(), magnitude, int(interleaved)
    for name, t in (("key_scale_stride", key_scale), ("value_scale_stride", value_scale)):
        setattr(a, name, int(t is not None and t.numel() > 1))
    return a


def append(key, value, key_cache, value_cache, slots, positions=None, frequencies=None, interleaved=False, magnitude=1.0, query=None, query_output=None,
           key_scale=None, value_scale=None, at_end=True):
    """hfrk_append_kv of CPU tensors (key None: hfrk_rotary), each in memory of its own; writes to the caches and to query_output."""
    m = Memory(at_end)
    written = [(t, m.copy(t)) for t in (key_cache, value_cache, query_output) if t is not None]
    at = {id(t): p for t, p in written}
    a = _append_args(lambda t: at[id(t)] if id(t) in at else m.copy(t), key, value, key_cache, value_cache, slots, positions, frequencies, interleaved, magnitude,
                     query, query_output, key_scale, value_scale)
    lib = _load()
    _run(lambda: lib.hfrk_append_kv(ctypes.byref(a), None))
    for t, p in written:
        storage = t.untyped_storage()
        ctypes.memmove(storage.data_ptr(), p - t.storage_offset() * t.element_size(), storage.nbytes())
    return query_output


def append_where_they_are(key, value, key_cache, value_cache, slots, positions=None, frequencies=None, interleaved=False, magnitude=1.0, query=None,
                          query_output=None, key_scale=None, value_scale=None) -> int:
    """The same on the tensors' own memory, which they may share; its status."""
    return _load().hfrk_append_kv(ctypes.byref(_append_args(lambda t: t.data_ptr(), key, value, key_cache, value_cache, slots, positions, frequencies, interleaved,
                                                            magnitude, query, query_output, key_scale, value_scale)), None)
