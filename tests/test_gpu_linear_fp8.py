"""dense.fp8_weight and dense.linear_fp8 on the MI355X against their definitions
in 64 bits: packing (bit for bit), products of one row to many, rows and columns
that end inside tiles, outputs in f32 and bf16, NaN, streams and captured calls.

Tolerance of a product: the products of two e4m3 values are exact; k of them are
added in f32, in some order, each addition off by 2^-24 of a partial sum that is at
most S = sum |x w|; two scales multiply (2 x 2^-24 of the result): |error| <= (k +
2) 2^-24 S, and half a step of the output's type.  bf16 results may come from the
8-bit matrix instruction, which adds eight consecutive products after cutting each to
a multiple of 2^-13 of the power of two of the largest: up to 7 x 2^-13 of that
one, so 7 x 2^-13 S more (and, each cut and rounding being its own, 2^-13 and 2^-8 /
sqrt(3) of the result in the 2-norm of many, checked beside it)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _randn(seed, shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).cuda()


def _rows(seed, m, k):
    """Rows in 8 bits: every magnitude of e4m3, each row with a scale of its own."""
    from zealot_amd import dense
    x = _randn(seed, (m, k), 30.0).clamp(-448, 448).to(FP8)
    return dense.Fp8Rows(x, 0.01 + _randn(seed + 1, (m,)).abs())


def _check(y, x, w, ws, out_dtype):
    xd, wd = x.data.double() * x.scales.double()[:, None], w.double() * ws.double()[:, None]
    want, most = xd @ wd.T, xd.abs() @ wd.abs().T
    tol = (xd.shape[1] + 2) * 2.0 ** -24 * most + (2.0 ** -8 if out_dtype == BF else 2.0 ** -24) * want.abs() * (1 + 2.0 ** -7)
    assert y.dtype == out_dtype and y.shape == want.shape
    if out_dtype == BF:
        tol += 7 * 2.0 ** -13 * most
        if want.numel() >= 4096:
            assert (y.double() - want).norm() <= (2.0 ** -8 / 3 ** 0.5 + 2.0 ** -13) * want.norm()
    off = (y.double() - want).abs() - tol
    assert (off <= 0).all(), (off.max(), off.argmax())


@pytest.mark.parametrize("n,k", [(1, 16), (64, 128), (65, 144), (100, 1000), (130, 4096), (3, 13)])
def test_packing(n, k):
    from zealot_amd import dense
    w = _randn(1, (n, k)).to(FP8)
    ws = _randn(2, (n,)).abs()
    p = dense.fp8_weight(w, ws)
    assert p.scales is ws and p.shape == (n, k)
    assert torch.equal(p.rowmajor().view(torch.uint8), w.view(torch.uint8))
    # what lies behind the rows and columns is zero
    total = p.data.view(torch.uint8).ne(0).sum()
    assert total == w.view(torch.uint8).ne(0).sum()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (70, 300), (128, 4096)])
def test_rounding_of_weights(n, k, dtype):
    """Scales max |w| / 448 (one division: a step), values between the roundings of w / s (1 -+ 2^-22)."""
    from zealot_amd import dense
    w = _randn(1, (n, k)).to(dtype)
    if n > 2:
        w[1] = 0
        w[2, k - 1] = float("nan")
    p = dense.fp8_weight(w)
    q, s = p.rowmajor(), p.scales
    fine = torch.tensor([i for i in range(n) if i != 2 or n <= 2], device="cuda")
    wd = w[fine].double()
    want = (wd.abs().amax(1) / 448).clamp(min=2.0 ** -126)
    assert ((s[fine].double() - want).abs() <= want * 2.0 ** -23).all()
    v, e = wd / want[:, None], 2.0 ** -22
    lo, hi = [(v * f).clamp(-448, 448).float().to(FP8).double() for f in (1 - e, 1 + e)]
    got = q[fine].double()
    assert ((got >= torch.minimum(lo, hi)) & (got <= torch.maximum(lo, hi))).all()
    if n > 2:
        assert torch.isnan(s[2]) and torch.isnan(q[2].float()).all()
        assert s[1] == 2.0 ** -126 and (q[1].float() == 0).all()


SIZES = [(1, 64, 128), (1, 4096, 4096), (2, 100, 16), (3, 1, 272), (7, 65, 144), (16, 192, 2048), (17, 130, 528), (33, 257, 1040), (48, 1000, 256),
         (64, 6144, 1024), (65, 200, 128), (100, 129, 400), (128, 128, 128), (129, 300, 4096), (200, 4096, 144), (257, 1030, 384), (513, 512, 2064),
         (4, 60000, 64)]


@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(m, n, k, out_dtype):
    from zealot_amd import dense
    x, w, ws = _rows(3, m, k), _randn(5, (n, k), 20.0).clamp(-448, 448).to(FP8), 0.01 + _randn(6, (n,)).abs()
    y = dense.linear_fp8(x, dense.fp8_weight(w, ws), out_dtype=out_dtype)
    _check(y, x, w, ws, out_dtype)


@pytest.mark.parametrize("m,n,k", [(4100, 4200, 256), (2049, 8192, 144), (300, 28672, 512), (1000, 9000, 16), (2300, 4100, 80), (700, 20000, 64),
                                   (1025, 7000, 1040), (900, 4160, 1472), (64, 4096, 14336), (40, 1000, 8192), (130, 2000, 6000), (256, 70, 16384),
                                   (2560, 4096, 208), (4000, 4030, 2000), (3900, 4030, 1040), (500, 28610, 2192),
                                   (300, 30001, 1072), (500, 30000, 1088), (4000, 4096, 640), (8200, 4100, 528)])
def test_large_products(m, n, k):
    from zealot_amd import dense
    x, w, ws = _rows(3, m, k), _randn(5, (n, k), 20.0).clamp(-448, 448).to(FP8), 0.01 + _randn(6, (n,)).abs()
    _check(dense.linear_fp8(x, dense.fp8_weight(w, ws)), x, w, ws, BF)


@pytest.mark.parametrize("m", [1, 5, 40, 64, 90, 300])
def test_every_output_is_written_and_nothing_else(m):
    from zealot_amd import dense
    n, k = 77, 160
    x, w, ws = _rows(3, m, k), _randn(5, (n, k)).to(FP8), _randn(6, (n,)).abs()
    for dtype in (BF, F32):
        buf = torch.full((m * n + 64,), 7.0, dtype=dtype, device="cuda")
        y = dense.linear_fp8(x, dense.fp8_weight(w, ws), out=buf[:m * n].view(m, n))
        _check(y, x, w, ws, dtype)
        assert (buf[m * n:] == 7).all()


@pytest.mark.parametrize("m", [1, 20, 64, 150, 600])
def test_nan_and_padding(m):
    """NaN stays in its row and its column; what lies behind a row of x is not taken for it (k % 128)."""
    from zealot_amd import dense
    n, k = 200, 208
    x, w, ws = _rows(3, m, k), _randn(5, (n, k)).to(FP8), _randn(6, (n,)).abs()
    # the buffer behind x and the rows' neighbours are NaN codes
    buf = torch.full((m * k + 4096,), 0x7f, dtype=torch.uint8, device="cuda")
    buf[:m * k] = x.data.view(torch.uint8).flatten()
    x = dense.Fp8Rows(buf[:m * k].view(FP8).view(m, k), x.scales)
    _check(dense.linear_fp8(x, dense.fp8_weight(w, ws)), x, w, ws, BF)
    w2 = w.clone()
    w2.view(torch.uint8)[9, 3] = 0x7f
    y = dense.linear_fp8(x, dense.fp8_weight(w2, ws))
    assert torch.isnan(y[:, 9]).all() and torch.isnan(y).sum() == m
    x2 = dense.Fp8Rows(x.data.clone(), x.scales.clone())
    x2.data.view(torch.uint8)[m - 1, k - 1] = 0xff
    y = dense.linear_fp8(x2, dense.fp8_weight(w, ws))
    assert torch.isnan(y[m - 1]).all() and torch.isnan(y).sum() == n
    x2 = dense.Fp8Rows(x.data, x.scales.clone())
    x2.scales[0] = float("nan")
    y = dense.linear_fp8(x2, dense.fp8_weight(w, ws))
    assert torch.isnan(y[0]).all() and torch.isnan(y).sum() == n


def test_outputs_past_2_32():
    """The last rows of an output of more than 2^32 values are those of a small call."""
    from zealot_amd import dense
    n, k = 16384, 16
    m = (1 << 32) // n + 300
    w, ws = _randn(5, (n, k)).to(FP8), _randn(6, (n,)).abs()
    p = dense.fp8_weight(w, ws)
    small = _rows(3, 300, k)
    x = dense.Fp8Rows(torch.zeros((m, k), device="cuda").to(FP8), torch.ones(m, device="cuda"))
    x.data[-300:], x.scales[-300:] = small.data, small.scales
    y = dense.linear_fp8(x, p)
    _check(y[-300:], small, w, ws, BF)
    assert (y[:300] == 0).all() and (y[m // 2:m // 2 + 300] == 0).all()


def test_rows_from_the_norm():
    """The 8-bit rows of a norm against a rounded weight: within the two roundings (2^-4 a value each) of the product
    of the values before them."""
    from zealot_amd import dense
    x, w, nw = _randn(1, (40, 1024)).bfloat16(), _randn(2, (300, 1024), 1 / 32).bfloat16(), _randn(3, (1024,)).bfloat16()
    y = dense.linear_fp8(dense.rms_norm_fp8(x, nw), dense.fp8_weight(w), out_dtype=F32)
    d = x.double()
    t = d * (d.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * nw.double()
    want = t @ w.double().T
    # a rounded value is off by 2^-4 of itself or half the smallest step, 2^-10 of a scale
    et = t.abs() * 2.0 ** -4 + (t.abs().amax(1, keepdim=True) / 448) * 2.0 ** -10
    ew = w.double().abs() * 2.0 ** -4 + (w.double().abs().amax(1, keepdim=True) / 448) * 2.0 ** -10
    tol = et @ w.double().abs().T + t.abs() @ ew.T + et @ ew.T
    assert ((y.double() - want).abs() <= tol * (1 + 2.0 ** -10)).all()
    # and, the roundings being of either sign, far nearer in the mean: 2^-4 / sqrt(3) a value at most, of two values
    assert (y.double() - want).norm() <= 2.0 ** -4 * (2 / 3) ** 0.5 * 1.05 * want.norm()


def test_streams_and_capture():
    from zealot_amd import dense
    n, k = 300, 512
    w, ws = _randn(5, (n, k)).to(FP8), _randn(6, (n,)).abs()
    p = dense.fp8_weight(w, ws)
    for m in (3, 50, 200):
        x = _rows(3, m, k)
        want = dense.linear_fp8(x, p)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = dense.linear_fp8(x, p, stream=side)
        side.synchronize()
        assert torch.equal(got, want)
        xs = dense.Fp8Rows(x.data.clone(), x.scales.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = dense.linear_fp8(xs, p)
        for i in range(3):
            xs.scales.copy_(x.scales * (i + 1))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, dense.linear_fp8(xs, p))
