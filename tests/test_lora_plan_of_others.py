"""dense.lora refuses a plan made for another number of adapters (CPU): with fewer rows
than adapters its tiles have the same shape, and rows whose adapter the weights do not
hold would be left out."""
import pytest
import torch

from zealot_amd import _lib, dense


def _plan(rows, adapters):
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dense.LoraPlan(z(rows), z(adapters + 1), z(_lib.lib().zk_lora_max_tiles(rows, adapters), 2))


@pytest.mark.parametrize("planned,held", [(100, 50), (50, 100), (4, 3), (2048, 1)])
def test_plans_of_other_adapters(planned, held):
    x, y = torch.zeros((3, 64)), torch.zeros((3, 32))
    a, b = torch.zeros((held, 8, 64)), torch.zeros((held, 32, 8))
    with pytest.raises(ValueError, match=f"plan is of {planned} adapters, the weights of {held}"):
        dense.lora(x, a, b, None, _plan(3, planned), y)
    with pytest.raises(ValueError, match="GPU"):  # (its own plan: on to the operands' device)
        dense.lora(x, a, b, None, _plan(3, held), y)
