"""Calls of so many rows that one launch would pass 2^32 threads, which the runtime counts in 32 bits: on the CPU, over the stand-in for the HIP runtime."""
import os
import subprocess
import sys

import pytest

from test_workspace_host import _PRELUDE, _fields, stand_in  # noqa: F401  (a fixture)

_CALLS = {
    "quantize_int8": "lib.hfrk_quantize_int8(1 << 20, None, 1 << 40, 1 << 44, rows, cols, _capi.BF16, 1)",
    "quantize_int8_static": "lib.hfrk_quantize_int8(1 << 20, 64, 1 << 40, None, rows, cols, _capi.BF16, 1)",
    "quantize_fp8": "lib.hfrk_quantize_fp8(1 << 20, None, 1 << 40, 1 << 44, rows, cols, _capi.BF16, 1)",
    "swiglu_dynamic_int8": "lib.hfrk_swiglu_dynamic_int8(1 << 20, 1 << 40, 1 << 44, rows, cols, _capi.BF16, 1)",
    "swiglu_dynamic": "lib.hfrk_swiglu_dynamic(1 << 20, 1 << 40, 1 << 44, None, rows, cols, 0, _capi.BF16, 1)",
}


@pytest.mark.parametrize("call", sorted(_CALLS))
def test_every_row_has_its_workgroup(call, stand_in):  # noqa: F811
    from hf_rocm_kernels import _capi
    code = _PRELUDE.format(package=os.path.dirname(_capi.__file__), stand_in=stand_in, fields=_fields()) + f"""
for rows, cols in ((1, 8), ((1 << 26) - 1, 8), ((1 << 26) + 5, 8), (1 << 27, 512), ((1 << 31) - 1, 8), (1 << 23, 4096), ((1 << 23) + 1, 8192)):
    stand_in.stand_in(0, 0)
    assert {_CALLS[call]} == _capi.SUCCESS, (rows, cols)
    assert stand_in.stand_in_groups() == rows and stand_in.stand_in_most_threads() < 1 << 32, (rows, cols, stand_in.stand_in_groups())
"""
    preload = ":".join(p for p in (stand_in, os.environ.get("LD_PRELOAD")) if p)
    subprocess.run([sys.executable, "-c", code], check=True, timeout=100, env=dict(os.environ, LD_PRELOAD=preload))
