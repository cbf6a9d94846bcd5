"""Products grouped by expert, and of int8 codes, on every tile shape that the cost models choose: ragged and empty groups, gathered rows, a part of a stage at the end
of k, rows that are no whole pieces, k shared between workgroups.  That each size runs on its shape is checked on the CPU, over the stand-in for the HIP runtime."""
import json
import os
import random
import re
import subprocess
import sys

import pytest
import torch

from hf_rocm_kernels import _capi
from hf_rocm_kernels.operators.int8_gemm import int8_gemm, reference_int8_gemm
from test_grouped_gemm_gpu import FP8, INT8, _close, _codes, _grouped, _magnitude, _scales
from test_workspace_host import _PRELUDE, _fields, stand_in  # noqa: F401  (a fixture)

# (experts, mean rows of a group, n, k) by (TM, TN, WM, WN, stages, workgroups a compute unit)
GROUPS = {
    (4, 2, 2, 4, 5, 1): [(16, 300, 2056, 16), (60, 301, 1030, 208), (60, 79, 1000, 784), (70, 159, 513, 784)],
    (2, 2, 4, 2, 3, 1): [(60, 200, 264, 2064), (70, 135, 257, 1296), (70, 128, 264, 1328), (60, 315, 130, 1296)],
    (2, 2, 2, 2, 5, 1): [(60, 12, 1000, 4112), (60, 12, 513, 5424), (60, 11, 1000, 2912)],
    (2, 1, 2, 2, 3, 2): [(5, 14, 8, 304), (3, 14, 101, 704), (3, 100, 264, 688)],
    (2, 1, 2, 4, 5, 2): [(60, 12, 520, 16), (33, 27, 1030, 32), (8, 300, 1000, 272), (60, 11, 257, 720), (60, 11, 264, 656), (8, 12, 2056, 688)],
}
# (m, n, k) of one weight by (those, waves that only load, whether k is shared between workgroups)
DENSE = {
    (4, 2, 2, 4, 5, 1, 0, False): [(1923, 4099, 16), (1296, 6000, 16), (1921, 4099, 336), (1307, 6000, 336)],
    (4, 2, 2, 4, 5, 1, 0, True): [(1008, 4099, 12752), (2028, 2056, 13296)],
    (2, 2, 4, 2, 3, 1, 0, False): [(1430, 4099, 144), (1437, 4104, 144)],
    (2, 2, 4, 2, 3, 1, 4, False): [(1434, 4099, 304), (1519, 4104, 272)],
    (2, 2, 4, 2, 3, 1, 4, True): [(436, 4099, 7696), (132, 6000, 14288)],
    (2, 2, 2, 2, 5, 1, 4, False): [(416, 4099, 1104), (418, 4104, 1072)],
    (2, 2, 2, 2, 5, 1, 4, True): [(198, 4099, 6672), (70, 6000, 12592)],
    (2, 1, 2, 2, 3, 2, 0, False): [(65, 101, 16), (300, 264, 144)],
    (2, 1, 2, 2, 3, 2, 4, False): [(68, 101, 304), (71, 264, 272)],
    (2, 1, 2, 2, 3, 2, 4, True): [(71, 4099, 7440), (66, 4104, 8080)],
    (1, 1, 2, 2, 8, 1, 4, False): [(70, 101, 400), (65, 264, 400)],
    (1, 1, 2, 2, 8, 1, 4, True): [(66, 101, 4080), (69, 264, 4240)],
}

_RUN = r"""
import json, re
class Name(ctypes.Structure):
    _fields_ = [("file", ctypes.c_char_p), ("base", ctypes.c_void_p), ("name", ctypes.c_char_p), ("address", ctypes.c_void_p)]

def numbers():  # of the kernel's template
    found = Name()
    assert ctypes.CDLL(None).dladdr(ctypes.c_void_p(stand_in.stand_in_kernel()), ctypes.byref(found)) and b"tiled_gemm_kernel" in found.name, found.name
    return [int(x) for x in re.findall(r"L[ib](\d+)E", found.name.decode())]

P, out = 1 << 40, []
for kind, *size in json.loads(sys.argv[1]):
    stand_in.stand_in(0, 0)
    if kind == "dense":
        m, n, k = size
        need = lib.hfrk_int8_gemm_workspace_bytes(m, n, k)
        assert lib.hfrk_int8_gemm(P, P, P, None, 0, P, 1, P, 1, m, n, k, k, _capi.BF16, P if need else None, need, 1) == _capi.SUCCESS
        out.append(numbers() + [need > 0])
    else:
        experts, mean, n, k = size
        args = _capi.GroupedArgs(a=P, rows=P, b=P, expert_stride=n * k, output=P, scale_a=P, scale_b=P, scale_b_expert_stride=n, offsets=P, scale_a_stride=1, scale_b_stride=1,
                                 b_stride=k, count=experts * mean, a_rows=experts * mean, experts=experts, n=n, k=k, type=_capi.INT8 if kind == "int8" else _capi.FP8_E4M3FN,
                                 dtype=_capi.BF16)
        assert lib.hfrk_grouped_gemm(ctypes.byref(args), 1) == _capi.SUCCESS
        out.append(numbers())
print("OUT", json.dumps(out))
"""


def _kernels(calls, stand_in):  # noqa: F811
    code = _PRELUDE.format(package=os.path.dirname(_capi.__file__), stand_in=stand_in, fields=_fields()) + _RUN
    preload = ":".join(p for p in (stand_in, os.environ.get("LD_PRELOAD")) if p)
    done = subprocess.run([sys.executable, "-c", code, json.dumps(calls)], check=True, timeout=100, env=dict(os.environ, LD_PRELOAD=preload), stdout=subprocess.PIPE, text=True)
    return json.loads(done.stdout.split("OUT ")[1])


def test_sizes_run_on_their_shapes(stand_in):  # noqa: F811
    """Template parameters: the shape's six, packed, waves that only load, int8, grouped, halves of stages."""
    calls, wanted = [], []
    for shape, sizes in GROUPS.items():
        for size in sizes:
            for kind in ("fp8", "int8"):
                calls.append((kind, *size))
                wanted.append((list(shape), kind == "int8", True, None))
    for (*shape, loaders, shared), sizes in DENSE.items():
        for size in sizes:
            calls.append(("dense", *size))
            wanted.append((shape, True, False, (loaders, shared)))
    for call, got, (shape, int8, grouped, rest) in zip(calls, _kernels(calls, stand_in), wanted):
        assert got[:6] == shape and got[8] == int8 and got[9] == grouped, (call, got)
        assert rest is None or (got[7], got[11]) == rest, (call, got)


def test_every_shape_of_groups_is_listed():
    with open(os.path.join(os.path.dirname(_capi.LIB_PATH), os.pardir, "csrc", "grouped_gemm.h")) as f:
        text = f.read()
    text = text[text.index("#define HFRK_GROUP_SHAPES"):text.index("#define HFRK_GROUP_ROW")]
    assert {tuple(map(int, row)) for row in re.findall(r"X\(\d, (\d), (\d), (\d), (\d), (\d), (\d)\)", text)} == set(GROUPS)


def _ragged(experts, mean, seed):
    """Sizes of that mean: some experts have none, some many rows."""
    rng = random.Random(seed)
    appeal = [0.0 if rng.random() < 0.15 else rng.lognormvariate(0.0, 1.0) for _ in range(experts)]
    appeal[rng.randrange(experts)] += 1.0
    left, sizes = experts * mean, []
    for e in range(experts):
        sizes.append(min(left, round(left * appeal[e] / sum(appeal[e:])) if sum(appeal[e:]) else 0))
        left -= sizes[-1]
    sizes[-1] += left
    assert sum(sizes) == experts * mean
    return sizes


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [FP8, INT8])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("experts,mean,n,k", [size for sizes in GROUPS.values() for size in sizes])
def test_groups(codes, gather, experts, mean, n, k):
    sizes = _ragged(experts, mean, n + k)
    _grouped(sizes, k, n, codes, torch.float16 if n % 16 else torch.bfloat16, gather, seed=experts + mean)
    even = [mean] * (experts - 1) + [mean - min(mean, 7)]  # the last rows are no group's
    _grouped(even, k, n, codes, torch.bfloat16, gather, seed=mean, front=2, behind=min(mean, 7) - 2)


@pytest.mark.gpu
@pytest.mark.parametrize("base", [None, "row", "full"])
@pytest.mark.parametrize("m,n,k", [size for sizes in DENSE.values() for size in sizes])
def test_one_weight(m, n, k, base):
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    dtype = torch.bfloat16 if base else torch.float16
    a, w = _codes(gen, (m, k), INT8), _codes(gen, (n, k), INT8)
    sa, sb = _scales(gen, m) / 16, _scales(gen, n)  # (within float16)
    add = {None: None, "row": torch.randn(n, generator=gen, device="cuda").to(dtype), "full": torch.randn((m, n), generator=gen, device="cuda").to(dtype)}[base]
    out = int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype)
    exact = reference_int8_gemm(a, w.t(), sa, sb, add)
    _close(out, exact, _magnitude(a, w, sa, sb), k, INT8, add)
    assert torch.equal(int8_gemm(a, w.t(), sa, sb, base=add, out_dtype=dtype), out)
    if base == "full":
        assert int8_gemm(a, w.t(), sa, sb, base=add, output=add) is add and torch.equal(add, out)
