"""What the compiler makes of the tiled kernels on groups and on int8 codes: the same orders as of the fp8 ones, and no registers in scratch memory."""
import re

import pytest

from test_kernel_assembly import _assembly, _instances


@pytest.mark.parametrize("source,count", [("tiled_int8.hip", 7), ("tiled_grouped_fp8.hip", 5), ("tiled_grouped_int8.hip", 5)])
def test_loads_read_no_scalar_that_a_vector_instruction_has_just_written(source, count, tmp_path):
    """The kernel's own wait states stand between the last v_readfirstlane that makes a buffer and the first load in inline assembly, and nothing makes one
    afterwards, gathered rows and a group's weight included."""
    instances = _instances(source, "tiled_gemm_kernel", tmp_path)
    assert len(instances) == count
    for name, body in instances.items():
        loads = [i for i, x in enumerate(body) if x.endswith(" lds")]
        waits = [i for i, x in enumerate(body) if x == "s_nop 4" and i < loads[0]]
        written = [i for i, x in enumerate(body) if x.startswith(("v_readfirstlane", "v_readlane"))]
        assert loads and waits, name
        assert not [i for i in written if waits[-1] < i < loads[-1]], name


@pytest.mark.parametrize("source", ["tiled_int8.hip", "tiled_grouped_fp8.hip", "tiled_grouped_int8.hip", "grouped_gemm.hip", "experts.hip"])
def test_registers_are_enough(source, tmp_path):
    sizes = [int(x) for x in re.findall(r"\.private_segment_fixed_size: (\d+)", "".join(_assembly(source, tmp_path)))]
    assert sizes and max(sizes) == 0, sizes


def test_row_split_kernel_on_int8_codes_keeps_its_registers(tmp_path):
    """As on fp8 codes: the loop of the 32-row instances fills all 256, at most one pair of registers lives in scratch; the scales are asked for with the first chunk."""
    sizes = [int(x) for x in re.findall(r"\.private_segment_fixed_size: (\d+)", "".join(_assembly("skinny_gemm_rows_int8.hip", tmp_path)))]
    assert len(sizes) == 20 and max(sizes) <= 8
    for name, body in _instances("skinny_gemm_rows_int8.hip", "skinny_gemm_rows_kernel", tmp_path).items():
        first = next(i for i, x in enumerate(body) if x.startswith("buffer_load_dwordx4") and " nt" in x)
        scale = next(i for i, x in enumerate(body) if x.startswith("global_load_dword "))
        assert 0 < scale - first < 60, (name, scale - first)


def test_kernel_that_splits_k_keeps_its_registers(tmp_path):
    sizes = [int(x) for x in re.findall(r"\.private_segment_fixed_size: (\d+)", "".join(_assembly("skinny_gemm_ksplit.hip", tmp_path)))]
    assert len(sizes) == 42 and max(sizes) == 0
