"""Registers of the kernels of a serving step (step tables, norms with rotation,
page bounds, scores, selection and sparse decode), read from the code objects of the
built library: none keeps registers in memory, and the waves a SIMD that their
comments count on fit its 512 registers."""
import pytest

from tests.test_kernel_resources import SIMD_VGPRS, _all, _alloc, _one, kernel_registers

OBJECTS = ["step_ops.o", "rope_ops.o", "sparse_ops.o", "paged_sparse.o"]


@pytest.mark.parametrize("obj", OBJECTS)
def test_nothing_spills(obj, tmp_path):
    regs = kernel_registers(obj, tmp_path)
    assert regs
    for name, (_, _, priv) in regs.items():
        assert priv == 0, f"{name} keeps {priv} bytes a lane in memory"


def _waves(v: int, a: int) -> int:
    return SIMD_VGPRS // _alloc(v + a)


def test_selection_fits_its_workgroups(tmp_path):
    """16 waves of a row are four on every SIMD."""
    for name, (v, a, _) in _all(kernel_registers("sparse_ops.o", tmp_path), "select_pages_kernelILi16E").items():
        assert _waves(v, a) >= 4, name


def test_waves_of_the_batch_kernels(tmp_path):
    """Rotation of 32 + 2 x 8 heads of 128 bf16: five waves a SIMD; sparse decode of bf16 and fp8 pools, heads of 128
    (template arguments: pool type, head size, parts of a query): three, as its LDS allows, with f32 queries too."""
    rope = kernel_registers("rope_ops.o", tmp_path)
    assert _waves(*_one(rope, "qk_norm_rope_kernelItLi3ELb0ELb0E")[:2]) >= 5
    sparse = kernel_registers("paged_sparse.o", tmp_path)
    for kind in (1, 2):
        for parts in (1, 3):
            assert _waves(*_one(sparse, f"sparse_mfma_kernelILi{kind}ELi128ELi{parts}E")[:2]) >= 3
