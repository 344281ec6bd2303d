"""dense.lora_plan and dense.lora on the MI355X: plans against a stable sort (whole
numbers: equal), products against their definition in 64 bits over types, ranks,
parts, lengths and layouts, rows without an adapter, adapters without rows, NaN,
streams and captured calls.

Tolerance of y + c b (a x), row by row.  a x adds k products of f32 (bf16 products
are exact in f32, f32 ones off by 2^-24) in some order: off by (k + 2) 2^-24 S1, S1 =
sum |a x|; c and an fp8 row's scale: 3 steps more.  bf16: those values are kept as
two bf16 of 8 bits each, of which the rest is 2^-9 x 2^-9 at most: 2^-17 with the
second's own rounding.  Then rank products, (rank + 2) 2^-24 of sum |b v|; y's
addition, a step, and y's rounding, half a step of its type (bf16 2^-8)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _randn(seed, shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _ids(seed, rows, adapters, run=1, without=0.2):
    rng = np.random.default_rng(seed)
    out = []
    while len(out) < rows:
        a = -1 if rng.random() < without else int(rng.integers(adapters))
        out += [a] * (1 if run == 1 else int(rng.integers(1, run + 1)))
    return np.array(out[:rows], np.int32)


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ plans

def _check_plan(ids, adapters, plan):
    valid = (ids >= 0) & (ids < adapters)
    order = np.argsort(np.where(valid, ids, adapters), kind="stable")[:valid.sum()]
    want = np.concatenate([order, -np.ones(len(ids) - len(order), np.int64)])
    assert np.array_equal(plan.order.cpu().numpy(), want)
    counts = np.bincount(ids[valid], minlength=adapters)
    offsets = np.concatenate([[0], counts.cumsum()])
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    tr = 16 if len(ids) <= 1024 else 32
    tiles = [(a | min(tr, offsets[a + 1] - p) << 16, p) for a in range(adapters) for p in range(offsets[a], offsets[a + 1], tr)]
    got = plan.tiles.cpu().numpy()
    assert len(tiles) <= len(got)
    assert got[:len(tiles)].tolist() == [list(t) for t in tiles] and (got[len(tiles):] == [-1, 0]).all()


@pytest.mark.parametrize("rows,adapters,run", [(1, 1, 1), (1, 2048, 1), (63, 3, 1), (64, 64, 1), (65, 5, 7), (256, 64, 1), (1000, 1, 1), (1024, 100, 1),
                                               (1025, 7, 40), (5000, 2048, 1), (32768, 500, 512), (40000, 33, 1), (3, 700, 1)])
@pytest.mark.parametrize("without", [0.0, 0.3, 1.0])
def test_plan(rows, adapters, run, without):
    from zealot_amd import dense
    ids = _ids(rows + adapters, rows, adapters, run, without)
    _check_plan(ids, adapters, dense.lora_plan(_dev(ids), adapters))


def test_plan_of_ids_that_name_no_adapter():
    from zealot_amd import dense
    ids = np.array([5, -1, 4, 2147483647, -2147483648, 0, 6, 4], np.int32)
    _check_plan(ids, 5, dense.lora_plan(_dev(ids), 5))
    empty = dense.lora_plan(_dev([]), 5)
    assert empty.order.numel() == 0 and empty.offsets.tolist() == [0] * 6


def test_plan_into_kept_tensors_and_captured():
    from zealot_amd import dense
    n, rows = 9, 200
    a, b = _ids(1, rows, n), _ids(2, rows, n, 30)
    ids = _dev(a)
    out = dense.lora_plan(ids, n)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dense.lora_plan(ids, n, out=out)
    for x in (b, a, b):
        ids.copy_(_dev(x))
        g.replay()
        torch.cuda.synchronize()
        _check_plan(x, n, out)


# --------------------------------------------------------------- products

def _case(seed, rows, adapters, rank, k, cols, dtype, x="same", run=1, without=0.2):
    from zealot_amd import dense
    ids = _ids(seed, rows, adapters, run, without)
    P, n = len(cols), sum(cols)
    xs = _randn(seed, (rows, k), dtype)
    if x == "fp8":
        xs = dense.Fp8Rows((xs.float() * 30).clamp(-448, 448).to(FP8), 0.01 + _randn(seed + 9, (rows,)).abs())
    return dict(ids=ids, x=xs, a=_randn(seed + 1, (adapters, P * rank, k), dtype, k ** -0.5), b=_randn(seed + 2, (adapters, n, rank), dtype),
                scales=_randn(seed + 3, (adapters,)).abs() + 0.5, y=_randn(seed + 4, (rows, n), dtype), cols=cols, rank=rank)


def _want(c, part=None):
    """(result, tolerance) in 64 bits; part: each column's."""
    from zealot_amd import dense
    ids, r, n = c["ids"], c["rank"], c["b"].shape[1]
    na, P = c["a"].shape[0], c["a"].shape[1] // r
    if part is None:
        part = np.repeat(np.arange(P), c["cols"])
    x = c["x"].data.double() * c["x"].scales.double()[:, None] if isinstance(c["x"], dense.Fp8Rows) else c["x"].double()
    y, bf = c["y"].double().clone(), c["b"].dtype == BF
    tol = torch.zeros_like(y)
    for i in range(na):
        rows = torch.tensor(np.flatnonzero(ids == i), device="cuda")
        if rows.numel() == 0:
            continue
        a, b, s = c["a"][i].double(), c["b"][i].double(), 1.0 if c["scales"] is None else float(c["scales"][i])
        v = s * (x[rows] @ a.T)
        ev = (x.shape[1] + 5) * 2.0 ** -24 * s * (x[rows].abs() @ a.abs().T) + (2.0 ** -17 if bf else 0) * v.abs()
        for p in range(P):
            at = torch.tensor(np.flatnonzero(part == p), device="cuda")
            w, vp, ep = b[at], v[:, p * r:(p + 1) * r], ev[:, p * r:(p + 1) * r]
            at = at[None, :].expand(rows.numel(), -1)
            to = rows[:, None].expand(-1, at.shape[1])
            y[to, at] += vp @ w.T
            tol[to, at] = ep @ w.abs().T + (r + 2) * 2.0 ** -24 * (vp.abs() @ w.abs().T)
            tol[to, at] += (2.0 ** -24 + (2.0 ** -8 if bf else 2.0 ** -24)) * (y[to, at].abs() + tol[to, at])
    return y, tol


def _check(c, got, part=None):
    want, tol = _want(c, part)
    none = (c["ids"] < 0) | (c["ids"] >= c["a"].shape[0])
    assert torch.equal(got[none], c["y"][none])
    off = (got.double() - want).abs() - tol
    assert (off <= 0).all(), (off.max(), off.argmax())


def _run(c, y=None, **kw):
    from zealot_amd import dense
    plan = dense.lora_plan(_dev(c["ids"]), c["a"].shape[0])
    y = c["y"].clone() if y is None else y
    kw.setdefault("parts", c["cols"] if len(c["cols"]) > 1 else None)
    assert dense.lora(c["x"], c["a"], c["b"], c["scales"], plan, y, **kw) is y
    return y


CASES = [(1, 1, 16, 4096, (4096,)), (64, 32, 16, 1024, (512, 128, 128)), (5, 3, 8, 64, (64,)), (17, 2, 1, 40, (30,)), (40, 7, 33, 129, (65, 7)),
         (100, 4, 64, 256, (100, 300)), (30, 2, 128, 512, (96,)), (20, 3, 256, 128, (64, 64)), (9, 2, 128, 96, (32, 32, 32, 32)), (33, 5, 5, 7, (3,)),
         (1200, 6, 16, 256, (192, 64, 64)), (1100, 3, 64, 128, (130,)), (2000, 40, 24, 72, (72,)), (1500, 2, 128, 64, (64, 64, 64, 64)),
         (1030, 2, 170, 64, (70, 10, 33)), (257, 16, 12, 136, (260,)), (3, 2000, 8, 32, (16,))]


@pytest.mark.parametrize("kind", ["bf16", "f32", "fp8"])
@pytest.mark.parametrize("rows,adapters,rank,k,cols", CASES)
def test_products(rows, adapters, rank, k, cols, kind):
    c = _case(rows, rows, adapters, rank, k, cols, F32 if kind == "f32" else BF, "fp8" if kind == "fp8" else "same", run=1 if rows < 1000 else 90)
    if rank * len(cols) > 512:
        pytest.skip("over the ranks of a call")
    _check(c, _run(c))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 50, 1100])
def test_column_slices_and_strided_rows(rows, dtype):
    """x and y as columns of larger tensors; the rest of those stays."""
    c = _case(7, rows, 4, 16, 128, (192,), dtype)
    big_x, big_y = _randn(1, (rows, 400), dtype), _randn(2, (rows, 500), dtype)
    for x0, y0 in ((0, 0), (64, 160), (13, 7)):  # (the last: off every alignment)
        c["x"], c["y"] = big_x[:, x0:x0 + 128], big_y[:, y0:y0 + 192].clone()
        buf = big_y.clone()
        _run(c, buf[:, y0:y0 + 192])
        _check(c, buf[:, y0:y0 + 192])
        rest = torch.ones(500, dtype=torch.bool)
        rest[y0:y0 + 192] = False
        assert torch.equal(buf[:, rest], big_y[:, rest])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("block,parts", [(16, 2), (64, 2), (128, 3), (8, 4), (100, 2)])
def test_parts_in_turn(block, parts, dtype):
    for rows in (20, 1100):
        c = _case(3, rows, 3, 16, 96, (block * parts * 2,), dtype)
        c["a"] = _randn(5, (3, parts * 16, 96), dtype, 0.1)
        part = np.arange(block * parts * 2) // block % parts
        _check(c, _run(c, parts=parts, part_block=block), part)


def test_without_scales_and_without_adapters():
    from zealot_amd import dense
    c = _case(3, 30, 4, 16, 64, (128,), BF)
    c["scales"] = None
    _check(c, _run(c))
    c["ids"][:] = -1
    assert torch.equal(_run(c), c["y"])
    none = dense.lora_plan(_dev([]), 4)
    y = c["y"][:0]
    assert dense.lora(c["x"][:0], c["a"], c["b"], None, none, y) is y


def test_nan_stays_in_its_row_and_part():
    """A part whose values overflow leaves the columns of the others, in blocks that hold both."""
    for rows in (20, 1100):
        c = _case(3, rows, 2, 16, 64, (40, 88), F32, without=0.0)
        clean = _run(c)
        c["a"] = c["a"].clone()
        c["a"][:, 16:] *= 1e38
        x = c["x"].clone()
        x[7, 3] = float("nan")
        c["x"] = x
        y = _run(c)
        assert torch.isnan(y[7]).all()
        keep = torch.arange(rows, device="cuda") != 7
        assert torch.equal(y[keep, :40], clean[keep, :40])
        assert not torch.isfinite(y[keep, 40:]).all()


def test_same_bits_every_time():
    c = _case(3, 700, 20, 16, 4096, (512, 128), BF)
    first = _run(c)
    for _ in range(3):
        assert torch.equal(_run(c), first)


def test_streams_workspaces_and_capture():
    """Two captured calls over one workspace that run in turn, replays on new inputs, another stream."""
    from zealot_amd import dense
    c = [_case(s, 60, 5, 16, 512, (256, 64), BF) for s in (1, 2)]
    plans = [dense.lora_plan(_dev(x["ids"]), 5) for x in c]
    ws = torch.empty(dense.lora_workspace_bytes(60, 5, 512, 16, 2, BF), dtype=torch.uint8, device="cuda")
    want = [_run(x) for x in c]
    ys, graphs = [torch.empty_like(w) for w in want], []
    for x, p, y in zip(c, plans, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y.copy_(x["y"])
            dense.lora(x["x"], x["a"], x["b"], x["scales"], p, y, parts=(256, 64), workspace=ws)
        graphs.append(g)
    for _ in range(3):
        for g, y, w in zip(graphs, ys, want):
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, w)
        ws.fill_(255)
    side = torch.cuda.Stream()
    y = c[0]["y"].clone()
    side.wait_stream(torch.cuda.current_stream())
    dense.lora(c[0]["x"], c[0]["a"], c[0]["b"], c[0]["scales"], plans[0], y, parts=(256, 64), stream=side)
    side.synchronize()
    assert torch.equal(y, want[0])


def test_rows_past_2_32():
    """y of more than 2^32 values: the rows of an adapter far behind."""
    from zealot_amd import dense
    n = 32768
    rows = (1 << 32) // n + 5
    ids = -np.ones(rows, np.int32)
    ids[[0, rows - 3, rows - 1]] = [1, 0, 1]
    x = torch.zeros((rows, 16), dtype=BF, device="cuda")
    y = torch.zeros((rows, n), dtype=BF, device="cuda")
    a, b = _randn(1, (2, 8, 16), BF), _randn(2, (2, n, 8), BF)
    pick = torch.tensor([0, rows - 3, rows - 1], device="cuda")
    x[pick] = _randn(3, (3, 16), BF)
    y[pick] = _randn(4, (3, n), BF)
    c = dict(ids=ids[[0, rows - 3, rows - 1]], x=x[pick], a=a, b=b, scales=None, y=y[pick].clone(), cols=(n,), rank=8)
    dense.lora(x, a, b, None, dense.lora_plan(_dev(ids), 2), y)
    _check(c, y[pick])
    assert not y[1:rows - 3].any()
