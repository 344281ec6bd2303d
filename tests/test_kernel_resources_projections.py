"""Registers of the 8-bit projections' and the adapters' kernels, read from the code
objects of the built library: none keeps registers in memory, and the waves that
their workgroups and comments count on fit a SIMD's 512 registers."""
import pytest

from tests.test_kernel_resources import SIMD_VGPRS, _all, _alloc, _one, kernel_registers

OBJECTS = ["fp8_rows.o", "fp8_gemm.o", "lora_ops.o"]


@pytest.mark.parametrize("obj", OBJECTS)
def test_nothing_spills(obj, tmp_path):
    regs = kernel_registers(obj, tmp_path)
    assert regs
    for name, (_, _, priv) in regs.items():
        assert priv == 0, f"{name} keeps {priv} bytes a lane in memory"


def _waves(v: int, a: int) -> int:
    return SIMD_VGPRS // _alloc(v + a)


def test_largest_tile_has_two_waves_a_simd(tmp_path):
    """256x256: eight waves a workgroup, one workgroup a CU."""
    for name, (v, a, _) in _all(kernel_registers("fp8_gemm.o", tmp_path), "fp8_gemm_big_kernel").items():
        assert _waves(v, a) >= 2, name


def test_waves_of_long_rows(tmp_path):
    """16 waves of a row (bf16, whole vectors) are four on every SIMD; SiLU's of up to 16384 values two workgroups a CU."""
    regs = kernel_registers("fp8_rows.o", tmp_path)
    for name, (v, a, _) in _all(regs, "ELi16ELi1E").items():
        assert _waves(v, a) >= 4, name
    assert _waves(*_one(regs, "fp8_rows_kernelILb0EtLi8ELi2ELi16ELi1E")[:2]) >= 8


def test_plan_fits_its_workgroup(tmp_path):
    """16 waves: four on every SIMD."""
    assert _waves(*_one(kernel_registers("lora_ops.o", tmp_path), "lora_plan_kernel")[:2]) >= 4
