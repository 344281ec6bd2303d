"""dense.rms_norm_fp8 and dense.silu_mul_fp8 on the MI355X against their
definitions in 64 bits: sizes from one value to the longest rows, selected rows,
residuals in place, column slices, operands off their alignment, rows of zeros
and rows that hold NaN or infinite values, streams and captured calls.

Tolerances.  The sum x + residual is one f32 addition and one rounding: equal.
A row's sum of squares adds at most 64 values a thread, then 6 + 16 partial sums,
of rounded squares: off by 87 steps of 2^-24 of itself, its root by half of that;
division, addition of eps, reciprocal root (4), the product with w, with the root
and the division by 448: 10 more.  So y and the scale are off by at most 60 x
2^-24 < 2^-18; a value lies between the roundings of y / s (1 - e) and (1 + e) with e
= 2^-17 (both of them move it).  SiLU: exp2
of a product off by 2^-24 of itself (|g| <= 6 here: 9 x 2^-24 in the exponent, 6 of the
result), 2 of its own, sum, reciprocal (2) and products, 13 steps: less than that."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
LEAST = 2.0 ** -126


def _randn(seed, shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _codes(v):
    return v.clamp(-448, 448).to(F32).to(FP8).double()


def _check(got, y):
    """got: Fp8Rows; y: rows in f64, finite."""
    q, s = got.data.double(), got.scales.double()
    want = (y.abs().amax(1) / 448).clamp(min=LEAST)
    assert ((s - want).abs() <= want * 2.0 ** -18).all(), ((s - want).abs() / want).max()
    v = y / want[:, None]
    e = 2.0 ** -17
    a, b = _codes(v * (1 - e)), _codes(v * (1 + e))
    assert ((q >= torch.minimum(a, b)) & (q <= torch.maximum(a, b))).all()


def _norm(x, w, eps, residual=None, rows=None):
    t = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if rows is not None:
        t = t[rows]
    d = t.double()
    return t, d * (d.pow(2).mean(1, keepdim=True) + eps).rsqrt() * w.double()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,dim", [(1, 4096), (3, 64), (7, 1), (2, 17), (5, 100), (33, 1000), (2, 4095), (9, 8192), (4, 16384), (300, 2048), (1, 520)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(rows, dim, dtype, residual):
    from zealot_amd import dense
    x, w = _randn(1, (rows, dim), dtype), (1 + 0.1 * _randn(2, (dim,))).to(dtype)
    r = _randn(3, (rows, dim), dtype) if residual else None
    t, y = _norm(x, w, 1e-6, r)
    got = dense.rms_norm_fp8(x, w, 1e-6, residual=r)
    if residual:
        got, kept = got
        assert torch.equal(kept, t)
    assert got.data.dtype == FP8 and got.data.shape == (rows, dim) and got.scales.shape == (rows,)
    _check(got, y)


def test_norm_of_the_longest_rows():
    from zealot_amd import dense
    for dtype, dim in ((BF, 32768), (F32, 16384)):
        x, w = _randn(1, (3, dim), dtype), _randn(2, (dim,), dtype)
        _check(dense.rms_norm_fp8(x, w), _norm(x, w, 1e-6)[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_selected_rows(dtype):
    from zealot_amd import dense
    x, r, w = _randn(1, (40, 256), dtype), _randn(2, (40, 256), dtype), _randn(3, (256,), dtype)
    rows = torch.tensor([39, 0, 7, 7, 12], device="cuda")
    got, kept = dense.rms_norm_fp8(x, w, residual=r, rows=rows)
    t, y = _norm(x, w, 1e-6, r, rows)
    assert torch.equal(kept, t)
    _check(got, y)
    # a row that is not there gives zeros, in a kept buffer too
    rows = torch.tensor([3, 40, -1, 1 << 40], device="cuda")
    out = dense.Fp8Rows(torch.full((4, 256), 1.0, device="cuda").to(FP8), torch.ones(4, device="cuda"))
    kept = torch.ones((4, 256), dtype=dtype, device="cuda")
    dense.rms_norm_fp8(x, w, residual=r, rows=rows, out=out, residual_out=kept)
    assert (out.data[1:].float() == 0).all() and (kept[1:] == 0).all() and (out.scales[1:] == LEAST).all()
    assert torch.equal(kept[0], _norm(x, w, 1e-6, r, rows[:1])[0][0])
    none = dense.rms_norm_fp8(x, w, rows=rows[:0])
    assert none.data.shape == (0, 256) and none.scales.shape == (0,)
    empty = dense.rms_norm_fp8(x[:0], w)
    assert empty.data.shape == (0, 256)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_residual_in_place(dtype):
    from zealot_amd import dense
    for which in ("residual", "x"):
        x, r, w = _randn(1, (50, 512), dtype), _randn(2, (50, 512), dtype), _randn(3, (512,), dtype)
        t, y = _norm(x, w, 1e-6, r)
        got, kept = dense.rms_norm_fp8(x, w, residual=r, residual_out=r if which == "residual" else x)
        assert torch.equal(r if which == "residual" else x, t)
        _check(got, y)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_off_alignment(dtype):
    """Operands whose addresses are only their elements' own."""
    from zealot_amd import dense
    n, dim = 6, 256
    off = lambda seed, shape: _randn(seed, (shape[0] * shape[-1] + 1,) if len(shape) > 1 else (shape[0] + 1,), dtype)[1:].view(shape)  # noqa: E731
    x, r, w = off(1, (n, dim)), off(2, (n, dim)), off(3, (dim,))
    t, y = _norm(x, w, 1e-6, r)
    got, kept = dense.rms_norm_fp8(x, w, residual=r)
    assert torch.equal(kept, t)
    _check(got, y)
    q = torch.zeros(n * dim + 1, device="cuda").to(FP8)[1:].view(n, dim)
    got = dense.rms_norm_fp8(_randn(1, (n, dim), dtype), w, out=dense.Fp8Rows(q, torch.empty(n, device="cuda")))
    _check(got, _norm(_randn(1, (n, dim), dtype), w, 1e-6)[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_zeros_nan_and_infinity(dtype):
    from zealot_amd import dense
    x, w = _randn(1, (6, 512), dtype), _randn(2, (512,), dtype)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 500] = float("inf")
    x[4, 0] = -float("inf")
    got = dense.rms_norm_fp8(x, w)
    fine = torch.tensor([0, 5], device="cuda")
    _check(dense.Fp8Rows(got.data[fine], got.scales[fine]), _norm(x, w, 1e-6, None, fine)[1])
    assert (got.data[1].float() == 0).all() and got.scales[1] == LEAST
    assert torch.isnan(got.scales[2:5]).all() and torch.isnan(got.data[2:5].float()).all()
    one = dense.silu_mul_fp8(x[:3], torch.ones_like(x[:3]))
    assert torch.isnan(one.scales[2]) and torch.isnan(one.data[2].float()).all() and torch.isfinite(one.scales[:2]).all()
    assert (one.data[1].float() == 0).all() and one.scales[1] == LEAST
    # values far below one: the scale stops at 2^-126
    tiny = torch.full((1, 64), 2.0 ** -120, device="cuda")
    got = dense.silu_mul_fp8(tiny, torch.ones_like(tiny))
    _check(got, torch.full((1, 64), 2.0 ** -121, device="cuda").double())
    assert got.scales[0] == LEAST


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,cols", [(1, 14336), (3, 1), (5, 33), (2, 4096), (17, 1408), (64, 11008), (2, 16384), (3, 4001)])
@pytest.mark.parametrize("fused", [False, True])
def test_silu(rows, cols, dtype, fused):
    from zealot_amd import dense
    gu = _randn(4, (rows, 2 * cols), dtype) * 3
    g, u = gu[:, :cols], gu[:, cols:]
    if not fused:
        g, u = g.contiguous(), u.contiguous()
    gd = g.double()
    _check(dense.silu_mul_fp8(g, u), gd / (1 + (-gd).exp()) * u.double())


def test_silu_far_out():
    """exp overflows or vanishes: the product is -0, 0 or the gate itself."""
    from zealot_amd import dense
    g = torch.tensor([[-200.0, -88.0, -1e30, 100.0, 200.0, 0.0, 1e-30, -1e-30]], device="cuda")
    u = torch.ones_like(g)
    gd = g.double()
    _check(dense.silu_mul_fp8(g, u), gd * torch.sigmoid(gd))


def test_rows_past_2_32():
    """Offsets that need more than 32 bits: the last rows are those of a small call."""
    from zealot_amd import dense
    cols = 32768
    rows = (1 << 32) // cols + 9
    g = torch.zeros((rows, cols), dtype=BF, device="cuda")
    g[-8:] = _randn(1, (8, cols), BF)
    got = dense.silu_mul_fp8(g, g)
    small = dense.silu_mul_fp8(g[-8:], g[-8:])
    assert torch.equal(got.data[-8:].view(torch.uint8), small.data.view(torch.uint8)) and torch.equal(got.scales[-8:], small.scales)
    assert (got.data[:-8].view(torch.uint8)[:: 1000] == 0).all()
    del got
    w = torch.ones(cols, dtype=BF, device="cuda")
    got = dense.rms_norm_fp8(g, w, rows=torch.arange(rows - 8, rows, device="cuda"))
    small = dense.rms_norm_fp8(g[-8:].contiguous(), w)
    assert torch.equal(got.data.view(torch.uint8), small.data.view(torch.uint8)) and torch.equal(got.scales, small.scales)


def test_streams_and_capture():
    from zealot_amd import dense
    x, r, w = _randn(1, (20, 1024), BF), _randn(2, (20, 1024), BF), _randn(3, (1024,), BF)
    want, kept = dense.rms_norm_fp8(x, w, residual=r)
    silu = dense.silu_mul_fp8(x, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, k2 = dense.rms_norm_fp8(x, w, residual=r, stream=side)
    side.synchronize()
    assert torch.equal(got.data.view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(k2, kept)
    xs = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, ka = dense.rms_norm_fp8(xs, w, residual=r)
        b = dense.silu_mul_fp8(xs, r)
    for i in range(3):
        xs.copy_(x if i != 1 else r)
        g.replay()
        torch.cuda.synchronize()
        e, ke = dense.rms_norm_fp8(xs, w, residual=r)
        f = dense.silu_mul_fp8(xs, r)
        for u, v in ((a, e), (b, f)):
            assert torch.equal(u.data.view(torch.uint8), v.data.view(torch.uint8)) and torch.equal(u.scales, v.scales)
        assert torch.equal(ka, ke)
    assert torch.equal(b.scales, silu.scales)
