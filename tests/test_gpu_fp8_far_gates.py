"""dense.silu_mul_fp8 of gates whose exp(-g) is near the end of f32's range: from -87.3
(there 1 / (1 + exp(-g)) is no normal number any more) to -88.7 the product is one, and
silu_mul has it; a row of such gates must not become zeros.  And gates near f32's smallest.

Tolerance: g log2(e) is between 126 and 128: its constant is off by 2^-25 of
itself and its rounding by half a step of 2^-17, 2^-18 each, times log(2); exp2, sum,
reciprocal and products 8 steps of 2^-24, and the reciprocal's quarter half a step of
2^-149, 2^-21 of itself at most (it is above 2^-129): below 2^-17.  A value lies between the
roundings of y / s (1 -+ 2^-16), since both y and s move."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _codes(v):
    return v.clamp(-448, 448).float().to(FP8).double()


def _check(got, y):
    q, s = got.data.double(), got.scales.double()
    want = y.abs().amax(1) / 448
    assert ((s - want).abs() <= want * 2.0 ** -17).all(), ((s - want).abs() / want).max()
    v, e = y / want[:, None], 2.0 ** -16
    a, b = _codes(v * (1 - e)), _codes(v * (1 + e))
    assert ((q >= torch.minimum(a, b)) & (q <= torch.maximum(a, b))).all()


def _silu(g):
    g = g.double()
    return g / (1 + (-g).exp())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols", [512, 333])
def test_rows_of_far_gates(dtype, cols):
    from zealot_amd import dense
    gen = torch.Generator().manual_seed(1)
    g = (-87.4 - 1.3 * torch.rand((9, cols), generator=gen)).to(dtype).clamp(min=-88.7).cuda()
    u = (torch.randn((9, cols), generator=gen) * 2.0 ** 100).to(dtype).cuda()
    _check(dense.silu_mul_fp8(g, u), _silu(g) * u.double())
    # the same products are silu_mul's
    assert (dense.silu_mul(g, u) != 0).float().mean() > 0.9


def test_gates_around_the_border():
    """One value each, so that each has a scale of its own."""
    from zealot_amd import dense
    g = torch.tensor([[-80.0], [-86.9], [-87.0], [-87.3], [-87.34], [-87.4], [-88.0], [-88.5], [-88.7]], device="cuda")
    u = torch.full_like(g, 2.0 ** 100)
    got = dense.silu_mul_fp8(g, u)
    _check(got, _silu(g) * u.double())
    assert (got.data.float() == -448).all()


def test_gates_beyond():
    """exp(-g) is no number of f32: -0, as silu_mul's; the other end is the gate itself."""
    from zealot_amd import dense
    g = torch.tensor([[-91.0, -1000.0, -3e38], [89.0, 500.0, 1e30]], device="cuda")
    u = torch.ones_like(g)
    got = dense.silu_mul_fp8(g, u)
    assert (got.data[0].view(torch.uint8) == 0x80).all() and (dense.silu_mul(g, u)[0] == 0).all()
    _check(dense.Fp8Rows(got.data[1:], got.scales[1:]), g[1:].double())


def test_gates_of_the_smallest_numbers():
    """Even multiples of 2^-149: half of one is a number, and what comes of it with an up of 2^126."""
    from zealot_amd import dense
    g = (2.0 * torch.arange(1, 257, dtype=torch.float64) * 2.0 ** -149).float()[None]
    u = torch.full_like(g, 2.0 ** 126)
    y = g.double() / 2 * 2.0 ** 126
    got = dense.silu_mul_fp8(g.cuda(), u.cuda())
    s = (y.amax() / 448).float()
    assert got.scales.item() == s.item()
    assert torch.equal(got.data.view(torch.uint8).cpu(), (y / s.double()).float().to(FP8).view(torch.uint8))
