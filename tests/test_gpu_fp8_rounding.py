"""q = e4m3(y / scale), to nearest even, bit for bit: what dense.fp8_weight,
silu_mul_fp8 and rms_norm_fp8 write for rows y that they compute exactly.

y is a power of two's worth of work away from the inputs in all three: a weight is
y itself; SiLU(64) = 64 in f32 (exp(-64) is far below a step of 1), so up = y / 64;
rows of 2s have the root 1 / 2 without an epsilon, so weight = y.  The rows hold every
value halfway between two of e4m3, times scales whose reciprocal f32 does not
have: y / scale is that halfway value and goes to the even neighbour, while y times
a rounded reciprocal may lie on either side of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _halfway():
    """256 values: every one halfway between two of e4m3 with both signs (five bits
    at most), the zeros, and 448, which fixes a row's scale."""
    v = torch.arange(0x7f, dtype=torch.uint8).view(FP8).float()
    t = (v[1:] + v[:-1]) / 2
    row = torch.cat([torch.tensor([448.0, -448.0, 0.0, -0.0]), t, -t])
    return row


def _scales(dtype):
    """f32: eight bits, bf16: three, so that they hold the products with five."""
    bits = 7 if dtype == F32 else 2
    s = 1 + torch.arange(1 << bits) / (1 << bits)
    return torch.cat([s * 2.0 ** e for e in (-9, 0, 4)])


def _codes(v):
    return v.to(FP8).view(torch.uint8)


def _equal(got, codes, scales):
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.data.view(torch.uint8).cpu(), codes)


def _rows_of(dtype):
    v, s = _halfway(), _scales(dtype)
    y = v[None, :] * s[:, None]
    assert torch.equal(y.to(dtype).float(), y) and torch.equal(y / s[:, None], v.expand_as(y))
    return y.to(dtype), _codes(v.expand_as(y)), s


@pytest.mark.parametrize("dtype", [BF, F32])
def test_weights(dtype):
    from zealot_amd import dense
    y, codes, s = _rows_of(dtype)
    p = dense.fp8_weight(y.cuda())
    _equal(dense.Fp8Rows(p.rowmajor(), p.scales), codes, s)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_any_weights(dtype):
    """Rows of any values: the host's quotients (f32, to nearest), rounded."""
    from zealot_amd import dense
    y = torch.randn((4000, 500), generator=torch.Generator().manual_seed(1)).to(dtype)
    s = y.float().abs().amax(1) / 448
    p = dense.fp8_weight(y.cuda())
    _equal(dense.Fp8Rows(p.rowmajor(), p.scales), _codes(y.float() / s[:, None]), s)


@pytest.mark.parametrize("cols", [256, 255])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu(dtype, cols):
    from zealot_amd import dense
    y, codes, s = _rows_of(dtype)
    y, codes = y[:, :cols].contiguous(), codes[:, :cols]
    up = (y.float() / 64).to(dtype).cuda()
    _equal(dense.silu_mul_fp8(torch.full_like(up, 64.0), up), codes, s)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm(dtype):
    from zealot_amd import dense
    y, codes, s = _rows_of(dtype)
    for i in range(0, len(s), 1 if dtype == BF else 16):
        x = torch.full((3, y.shape[1]), 2.0, dtype=dtype, device="cuda")
        _equal(dense.rms_norm_fp8(x, y[i].cuda(), 0.0), codes[i].expand(3, -1), s[i].expand(3))
