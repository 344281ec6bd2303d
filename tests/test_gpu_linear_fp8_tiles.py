"""dense.linear_fp8 on the MI355X on every tile that a call may take, k whole and split
(sizes of fp8_tiles.py), in both result types, against 64 bits with the tolerances of
test_gpu_linear_fp8.py; 9 to 16 rows of many columns; the decode batch's projections;
captured calls with split k that share a workspace."""
import pytest
import torch

from tests.fp8_tiles import SIZES, choose, stream
from tests.test_gpu_linear_fp8 import BF, F32, FP8, _check, _randn, _rows

pytestmark = pytest.mark.gpu


def _weight(n, k):
    return _randn(5, (n, k), 20.0).clamp(-448, 448).to(FP8), 0.01 + _randn(6, (n,)).abs()


def _product(m, n, k, dtype):
    from zealot_amd import dense
    x, (w, ws) = _rows(3, m, k), _weight(n, k)
    _check(dense.linear_fp8(x, dense.fp8_weight(w, ws), out_dtype=dtype), x, w, ws, dtype)


@pytest.mark.parametrize("tile,splits,m,n,k", SIZES["bfloat16"])
def test_bf16(tile, splits, m, n, k):
    _product(m, n, k, BF)


@pytest.mark.parametrize("tile,splits,m,n,k", SIZES["float32"])
def test_f32(tile, splits, m, n, k):
    _product(m, n, k, F32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kernel,m,n,k", [("2x4", 9, 5003, 272), ("2x4", 16, 16320, 1040), ("4x4", 11, 16390, 528), ("4x4", 16, 28672, 4096), ("1x4", 8, 5003, 1040),
                                          ("1x8", 13, 4000, 2064)])
def test_up_to_16_rows(kernel, m, n, k, dtype):
    assert stream(m, n) == kernel
    _product(m, n, k, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k", [(256, 4096, 14336), (256, 28672, 4096), (256, 6144, 4096), (128, 4096, 14336), (512, 4096, 14336)])
def test_decode_batches(m, n, k, dtype):
    _product(m, n, k, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k", [(20, 33, 8352), (66, 2147, 11808)])
def test_captured_calls_that_share_a_workspace(m, n, k, dtype):
    """Two graphs, each with a split product through one workspace, replayed in turn on new scales."""
    from zealot_amd import dense
    assert choose(m, n, k, dtype == F32)[1] > 1
    size = dense.linear_fp8_workspace_bytes(m, n, k, dtype)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    weights = [dense.fp8_weight(_randn(s, (n, k), 20.0).clamp(-448, 448).to(FP8), _randn(s + 1, (n,)).abs()) for s in (5, 7)]
    rows = [_rows(s, m, k) for s in (3, 9)]
    first = [r.scales.clone() for r in rows]
    ys = [torch.empty((m, n), dtype=dtype, device="cuda") for _ in rows]
    graphs = []
    for x, w, y in zip(rows, weights, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dense.linear_fp8(x, w, out=y, workspace=ws)
        graphs.append(g)
    for i in range(3):
        for g, x, w, y, s in zip(graphs, rows, weights, ys, first):
            x.scales.copy_(s * (i + 1))
            y.fill_(-1)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, dense.linear_fp8(x, w, out_dtype=dtype))
        ws.fill_(255)  # (NaN: nothing of an earlier call is used)
    _check(ys[0], rows[0], weights[0].rowmajor(), weights[0].scales, dtype)


@pytest.mark.parametrize("m,n,k", [(400, 25652, 416), (420, 25600, 464), (2100, 6100, 528), (2100, 6100, 592)])
def test_nan_rows_next_to_others_in_the_largest_tile(m, n, k):
    """k ends inside the last 128 columns, in their first or second half: what the tile
    reads there are the next row's values, here NaN."""
    from zealot_amd import dense
    assert choose(m, n, k, False)[0] == "256x256" and k % 128 in (16, 32, 80)
    x, (w, ws) = _rows(3, m, k), _weight(n, k)
    buf = torch.full((m * k + 4096,), 0x7f, dtype=torch.uint8, device="cuda")
    codes = buf[:m * k].view(m, k)
    codes.copy_(x.data.view(torch.uint8))
    codes[1::2] = 0x7f
    y = dense.linear_fp8(dense.Fp8Rows(codes.view(FP8), x.scales), dense.fp8_weight(w, ws))
    assert torch.isnan(y[1::2]).all()
    _check(y[::2], dense.Fp8Rows(x.data[::2], x.scales[::2]), w, ws, BF)
