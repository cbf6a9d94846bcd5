"""Norms of so many rows that one launch would pass 2^32 threads: on the CPU, over the stand-in for the HIP runtime, which also keeps the pointers that every launch
gets."""
import os
import subprocess
import sys

import pytest

from test_workspace_host import _PRELUDE, _STAND_IN, _STRUCT, _fields

_KEEP = """
static uint64_t kept[256][6], kept_groups[256];
uint64_t stand_in_pointer(int launch, int i) { return kept[launch][i]; }
uint64_t stand_in_groups_of(int launch) { return kept_groups[launch]; }
int hipLaunchKernel("""

# Calls of `rows` rows of `cols`, and of each launch's six first arguments, all pointers: what a row moves it by.
_X, _RES, _W, _OUT, _S, _NEXT = ("%d << 48" % i for i in range(1, 7))
_CALLS = {
    "residual_rms_dynamic": (f"lib.hfrk_residual_rms_dynamic({_X}, {_RES}, {_W}, 1e-5, {_OUT}, {_S}, {_NEXT}, rows, cols, 24, _capi.BF16, 1)",
                             f"(({_X}, 2 * cols), ({_RES}, 2 * cols), ({_W}, 0), ({_OUT}, cols), ({_S}, 4), ({_NEXT}, 48))"),
    "residual_rms_fp8": (f"lib.hfrk_residual_rms({_X}, {_RES}, {_W}, {_S}, 1e-5, {_OUT}, {_NEXT}, rows, cols, 24, _capi.F16, _capi.FP8_E4M3FN, 0, 0, 1)",
                         f"(({_X}, 2 * cols), ({_RES}, 2 * cols), ({_W}, 0), ({_S}, 0), ({_OUT}, cols), ({_NEXT}, 48))"),
    "residual_rms_16_bit": (f"lib.hfrk_residual_rms({_X}, {_RES}, {_W}, None, 1e-5, {_OUT}, {_NEXT}, rows, cols, 24, _capi.BF16, _capi.BF16, 256, 0, 1)",
                            f"(({_X}, 2 * cols), ({_RES}, 2 * cols), ({_W}, 0), (0, 0), ({_OUT}, 2 * cols), ({_NEXT}, 48))"),
    "residual_rms_by_elements": (f"lib.hfrk_residual_rms({_X}, {_RES}, {_W}, {_S}, 1e-5, {_OUT}, {_NEXT}, rows, cols, 24, _capi.BF16, _capi.BF16, 0, 1, 1)",
                                 f"(({_X}, 2 * cols), ({_RES}, 2 * cols), ({_W}, 0), ({_S}, 0), ({_OUT}, 2 * cols), ({_NEXT}, 48))"),
}


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    directory = tmp_path_factory.mktemp("stand_in")
    source, library = os.path.join(directory, "stand_in.c"), os.path.join(directory, "libstand_in.so")
    text = (_STAND_IN % _STRUCT).replace("int hipLaunchKernel(", _KEEP, 1)
    text = text.replace("    ++launches;", "    if (launches < 256) {\n        kept_groups[launches] = grid;\n"
                        "        for (int i = 0; i < 6; ++i) kept[launches][i] = *(uint64_t*)args[i];\n    }\n    ++launches;", 1)
    with open(source, "w") as f:
        f.write(text)
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", source, "-o", library], check=True)
    return library


@pytest.mark.parametrize("call", sorted(_CALLS))
def test_every_row_has_its_workgroup_and_its_memory(call, stand_in):
    from hf_rocm_kernels import _capi
    run, pointers = _CALLS[call]
    code = _PRELUDE.format(package=os.path.dirname(_capi.__file__), stand_in=stand_in, fields=_fields()) + f"""
for name in ("pointer", "groups_of"):
    getattr(stand_in, "stand_in_" + name).restype = ctypes.c_uint64
for rows, cols in ((1, 8), (70, 4096), ((1 << 26) - 1, 8), (1 << 26, 8), ((1 << 26) + 5, 8), (1 << 27, 512), ((1 << 31) - 1, 8), (1 << 23, 4096), ((1 << 23) + 1, 8192)):
    stand_in.stand_in(0, 0)
    assert {run} == _capi.SUCCESS, (rows, cols)
    first = 0
    for launch in range(stand_in.stand_in_launches()):
        for i, (start, step) in enumerate({pointers}):
            assert stand_in.stand_in_pointer(launch, i) == start + first * step, (rows, cols, launch, i)
        first += stand_in.stand_in_groups_of(launch)
    assert first == rows and stand_in.stand_in_most_threads() < 1 << 32, (rows, cols, first)
"""
    preload = ":".join(p for p in (stand_in, os.environ.get("LD_PRELOAD")) if p)
    subprocess.run([sys.executable, "-c", code], check=True, timeout=100, env=dict(os.environ, LD_PRELOAD=preload))
