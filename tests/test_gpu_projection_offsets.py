"""8-bit products and adapters whose weights, rows or results pass 2^31 elements: what
lies at the start, around element 2^31 and 2^32 and at the end, against 64 bits.  Bars:
bf16's half step; for the products 7 x 2^-13 of the sum of magnitudes and, of an f32
sum of k terms, k + 2 steps of 2^-24; for the adapters those steps of both sums and the
2^-17 to which values between them are held."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _filled(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda") * scale)
    return t


def _some(rows, cols):
    """Rows at the start, where element 2^31 and 2^32 lie, and at the end."""
    want = {0, 1, rows - 2, rows - 1}
    for p in (1 << 31, 1 << 32):
        want |= {p // cols - 1, p // cols, p // cols + 1}
    return torch.tensor(sorted(r for r in want if 0 <= r < rows), device="cuda")


@pytest.mark.parametrize("m,n,k", [(160000, 28672, 128), (160000, 28672, 640), (5, 1100000, 4096), (40, 1100000, 4096), (20, 300, 4194304)])
def test_products(m, n, k):
    """Rows of y, of the weight, and a k of 2^22."""
    from zealot_amd import dense
    x = dense.Fp8Rows(_filled((m, k), FP8, 1), 0.5 + torch.rand(m, device="cuda"))
    w, ws = _filled((n, k), FP8, 2), 0.5 + torch.rand(n, device="cuda")
    y = dense.linear_fp8(x, dense.fp8_weight(w, ws))
    rows, cols = _some(m, n), torch.unique(torch.cat([_some(n, k), torch.arange(0, n, max(1, n // 97), device="cuda")]))
    xd = x.data.view(torch.uint8)[rows].view(FP8).double() * x.scales[rows].double()[:, None]
    wd = w.view(torch.uint8)[cols].view(FP8).double() * ws[cols].double()[:, None]
    want, most = xd @ wd.T, xd.abs() @ wd.abs().T
    # the f32 sums' own rounding: a chain of k / 8 additions at most
    off = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + (7 * 2.0 ** -13 + (k + 2) * 2.0 ** -24) * most
    assert ((y[rows][:, cols].double() - want).abs() <= off).all()


@pytest.mark.parametrize("T,adapters,k,n,rank", [(1100000, 3, 4096, 4104, 16), (64, 2048, 8192, 8192, 160)])
def test_adapters(T, adapters, k, n, rank):
    """Rows of x and y, and adapters whose A and B pass 2^31 elements."""
    from zealot_amd import dense
    x, y = _filled((T, k), BF, 1), _filled((T, n), BF, 2)
    a, b = _filled((adapters, rank, k), BF, 3, k ** -0.5), _filled((adapters, n, rank), BF, 4, rank ** -0.5)
    ids = torch.randint(-1, adapters, (T,), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    ids[-1] = adapters - 1
    ids[0] = adapters - 2
    rows = torch.unique(torch.cat([_some(T, k), _some(T, n)]))
    before = y[rows].double()
    dense.lora(x, a, b, None, dense.lora_plan(ids, adapters), y)
    for i, t in enumerate(rows.tolist()):
        id_, got = int(ids[t]), y[t].double()
        if id_ < 0:
            assert torch.equal(got, before[i])
            continue
        A, B, xd = a[id_].double(), b[id_].double(), x[t].double()
        want = before[i] + B @ (A @ xd)
        off = ((k + rank + 8) * 2.0 ** -24 + 2.0 ** -17) * (B.abs() @ (A.abs() @ xd.abs())) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8)
        assert ((got - want).abs() <= off).all(), t
