"""dense.qk_norm_rope and ops.qk_norm_rope_append on the MI355X against the
formulas in 64 bits.

Tolerances.  With u = 2^-24: the sum of squares is of positive terms in at most
24 rounded additions, so the norm's factor is off by at most (24 + 2) / 2 u and
rsqrt's 2 u, the products by x and w add 2 u, the rotation's products and sum 2 u
of |y_a| + |y_b| (cosines and sines are at most 1): below 20 u (|y_a| + |y_b|).
Then a rounding to the output's type: half a step, 2^-8 of the value in bf16, 2^-4
in e4m3 (2^-10 below its normal range)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def _inputs(seed, T, H, Hkv, D, dtype, fused=True, weights=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, (H + 2 * Hkv) * D, generator=g).to(dtype).cuda()
    if not fused:
        q, k, v = [t.contiguous() for t in x.split((H * D, Hkv * D, Hkv * D), 1)]
    else:
        q, k, v = x.split((H * D, Hkv * D, Hkv * D), 1)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() if weights else None for _ in range(2)]
    return q.unflatten(1, (H, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, D)), w


def _reference(x, w, pos, table, interleaved, eps=1e-6):
    """(rotated rows, the tolerance's |y_a| + |y_b|) in 64 bits, on the CPU."""
    x = x.double().cpu()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double().cpu()
    y, mag = x.clone(), x.abs()
    if table is not None:
        table, pos = table.double().cpu(), pos.cpu().long()
        half = table.shape[1] // 2
        ok = (pos >= 0) & (pos < table.shape[0])
        cs = table[pos.clamp(0, table.shape[0] - 1)]
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = cs[:, i, None], cs[:, half + i, None]
            y[..., a] = x[..., a] * c - x[..., b] * s
            y[..., b] = x[..., b] * c + x[..., a] * s
            mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
        y[~ok] = 0
        mag[~ok] = 0
    return y, mag


def _close(got, ref, mag, dtype):
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= 20 * U * mag * (1 + HALF[dtype]) + HALF[dtype] * ref.abs() + 1e-37).all()), float(err.max())


def _positions(seed, T, most):
    pos = torch.randint(0, most, (T,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    return pos.cuda()


SHAPES = [(1, 32, 8, 128, 128), (37, 32, 8, 128, 128), (300, 4, 4, 64, 64), (5, 16, 2, 128, 64), (9, 6, 3, 96, 96), (9, 5, 1, 96, 32),
          (4, 3, 3, 256, 256), (3, 2, 1, 512, 512), (3, 2, 1, 1024, 1024), (7, 4, 2, 32, 32), (6, 3, 1, 80, 40), (6, 3, 1, 34, 30),
          (5, 2, 2, 2, 2), (6, 4, 1, 128, 8), (2000, 8, 2, 128, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,Hkv,D,rot", SHAPES)
def test_against_the_formula(T, H, Hkv, D, rot, interleaved, dtype):
    from zealot_amd import dense
    q, k, _, (wq, wk) = _inputs(T + D, T, H, Hkv, D, dtype)
    table = dense.rope_table(700, rot, 10000.0)
    pos = _positions(3, T, 700)
    qo, ko = dense.qk_norm_rope(q, k, pos, table, wq, wk, interleaved=interleaved)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        assert got.is_contiguous() and got.dtype == dtype
        _close(got, *_reference(x, w, pos, table, interleaved), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,which", [(128, (True, False)), (128, (False, True)), (128, (False, False)), (34, (False, True))])
def test_norms_alone_and_left_out(D, which, dtype):
    from zealot_amd import dense
    q, k, _, w = _inputs(11, 21, 8, 2, D, dtype)
    wq, wk = [x if on else None for x, on in zip(w, which)]
    table, pos = dense.rope_table(100, D), _positions(4, 21, 100)
    for tab, p in ((table, pos), (None, None)):
        qo, ko = dense.qk_norm_rope(q, k, p, tab, wq, wk, eps=1e-3)
        _close(qo, *_reference(q, wq, p, tab, False, 1e-3), dtype)
        _close(ko, *_reference(k, wk, p, tab, False, 1e-3), dtype)


def test_far_positions_keep_their_phase():
    """A table of a million positions: its rows against angles in 64 bits."""
    from zealot_amd import dense
    table = dense.rope_table(1 << 20, 64, 500000.0)
    p = torch.tensor([0, 1, 131071, (1 << 20) - 1])
    freq = 500000.0 ** (-np.arange(0, 64, 2) / 64)
    angle = p.numpy()[:, None].astype(np.float64) * freq
    want = np.concatenate([np.cos(angle), np.sin(angle)], 1)
    # angles below 2^20 in 64 bits: off by 2^-33 at most, then half a step of f32
    assert np.abs(table[p.cuda()].cpu().numpy() - want).max() <= U + 2.0 ** -32


@pytest.mark.parametrize("D", [128, 34])
def test_positions_outside_the_table_give_zero_rows(D):
    from zealot_amd import dense
    q, k, _, (wq, wk) = _inputs(5, 6, 4, 2, D, torch.bfloat16)
    pos = torch.tensor([0, -1, 99, 100, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    table = dense.rope_table(100, D)
    qo, ko = dense.qk_norm_rope(q, k, pos, table, wq, wk)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        _close(got, *_reference(x, w, pos, table, False), torch.bfloat16)
        assert bool((got[[1, 3, 4, 5]] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,interleaved", [(128, False), (128, True), (34, False)])
def test_in_place_in_the_fused_buffer(D, interleaved, dtype):
    from zealot_amd import dense
    q, k, v, (wq, wk) = _inputs(6, 50, 8, 2, D, dtype)
    table, pos = dense.rope_table(64, D), _positions(6, 50, 64)
    want = dense.qk_norm_rope(q, k, pos, table, wq, wk, interleaved=interleaved)
    kept = v.clone()
    got = dense.qk_norm_rope(q, k, pos, table, wq, wk, interleaved=interleaved, q_out=q, k_out=k)
    assert got[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)


def test_operands_off_their_alignment_and_odd_strides():
    from zealot_amd import dense
    T, H, Hkv, D = 20, 4, 2, 64
    q, k, _, (wq, wk) = _inputs(7, T, H, Hkv, D, torch.bfloat16, fused=False)
    table, pos = dense.rope_table(64, D), _positions(7, T, 64)
    want = dense.qk_norm_rope(q, k, pos, table, wq, wk)
    for pad in (1, 3, 8):
        buf = torch.zeros(T, (H + Hkv) * D + pad, dtype=torch.bfloat16, device="cuda")
        q2, k2 = buf[:, pad:pad + H * D].unflatten(1, (H, D)), buf[:, pad + H * D:].unflatten(1, (Hkv, D))
        q2.copy_(q)
        k2.copy_(k)
        got = dense.qk_norm_rope(q2, k2, pos, table, wq, wk)
        for a, b, x, w in ((got[0], want[0], q, wq), (got[1], want[1], k, wk)):
            _close(a, *_reference(x, w, pos, table, False), torch.bfloat16)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite_stay_in_their_head(value):
    from zealot_amd import dense
    q, k, _, (wq, wk) = _inputs(8, 3, 4, 2, 128, torch.bfloat16)
    table, pos = dense.rope_table(64, 128), _positions(8, 3, 64)
    want, _ = dense.qk_norm_rope(q, k, pos, table, wq, wk)
    q[1, 2, 5] = value
    got, _ = dense.qk_norm_rope(q, k, pos, table, wq, wk)
    assert not bool(torch.isfinite(got[1, 2]).all())
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)


def _pools(nb, Hkv, bs, D, kind):
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}[kind]
    return [torch.full((nb, Hkv, bs, D), 3.0, device="cuda").to(t) for _ in range(2)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,Hkv,D,bs", [(1, 32, 8, 128, 16), (70, 8, 2, 64, 16), (33, 5, 1, 96, 16), (20, 4, 2, 34, 8), (3000, 4, 2, 128, 16)])
def test_with_the_kv_write(T, H, Hkv, D, bs, dtype, kind):
    from zealot_amd import dense, ops
    q, k, v, (wq, wk) = _inputs(T + bs, T, H, Hkv, D, dtype)
    rot = D // 2 // 2 * 2
    table, pos = dense.rope_table(500, rot), _positions(9, T, 500)
    nb = T // bs + 3
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(1))[:T]
    slots[::7] = -1
    if T > 2:
        slots[2] = nb * bs  # past the pool: skipped like a negative one
    kp, vp = _pools(nb, Hkv, bs, D, kind)
    scales = {}
    if kind == "fp8":
        g = torch.Generator().manual_seed(2)
        scales = dict(k_scales=(0.01 + 0.02 * torch.rand(3, Hkv, generator=g)).cuda(), v_scales=(0.01 + 0.02 * torch.rand(3, Hkv, generator=g)).cuda(),
                      token_row=(torch.arange(T, dtype=torch.int32) % 3).cuda())
    qo = ops.qk_norm_rope_append(kp, vp, q, k, v, pos, slots.cuda(), table, wq, wk, **scales)
    _close(qo, *_reference(q, wq, pos, table, False), dtype)
    ref_k = _reference(k, wk, pos, table, False)
    live = (slots >= 0) & (slots < nb * bs)
    for pool, (ref, mag), sc in ((kp, ref_k, "k_scales"), (vp, (v.double().cpu(), v.double().cpu().abs()), "v_scales")):
        rows = pool.float().double().cpu().transpose(1, 2).reshape(nb * bs, Hkv, D)
        got, ref, mag = rows[slots[live]], ref[live], mag[live]
        if kind == "fp8":
            s = scales[sc].double().cpu()[scales["token_row"].cpu().long()][live][:, :, None]
            ref, mag = ref / s, mag / s
            err = (got - ref.clamp(-448, 448)).abs()
            # the reciprocal of the scale and the product: 2 u more
            assert bool((err <= 24 * U * mag * 1.0625 + torch.maximum(ref.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10))).all())
        else:
            out = {"f32": torch.float32, "bf16": torch.bfloat16}[kind]
            err = (got - ref).abs()
            assert bool((err <= 20 * U * mag * (1 + HALF[out]) + HALF[out] * ref.abs() + 1e-37).all())
        other = torch.ones(nb * bs, dtype=torch.bool)
        other[slots[live]] = False
        assert bool((rows[other] == 3.0).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D", [(20, 4, 96), (64, 8, 128), (32, 32, 128), (16, 8, 64), (40, 2, 256)])
def test_many_tokens_of_many_heads(H, Hkv, D, dtype, interleaved):
    """Every number of heads a lane and of waves a token, past the last whole group of tokens."""
    from zealot_amd import dense, ops
    T = 2100
    q, k, v, (wq, wk) = _inputs(T + D, T, H, Hkv, D, dtype)
    table, pos = dense.rope_table(500, D), _positions(5, T, 500)
    kp, vp = _pools(140, Hkv, 16, D, "f32" if dtype == torch.float32 else "bf16")
    slots = torch.randperm(140 * 16, generator=torch.Generator().manual_seed(3))[:T]
    qo = ops.qk_norm_rope_append(kp, vp, q, k, v, pos, slots.cuda(), table, wq, wk, interleaved=interleaved)
    _close(qo, *_reference(q, wq, pos, table, interleaved), dtype)
    rows = [p.transpose(1, 2).reshape(-1, Hkv, D)[slots.cuda()] for p in (kp, vp)]
    _close(rows[0], *_reference(k, wk, pos, table, interleaved), dtype)
    assert torch.equal(rows[1], v)
    q2, k2 = dense.qk_norm_rope(q, k, pos, table, wq, wk, interleaved=interleaved)
    _close(q2, *_reference(q, wq, pos, table, interleaved), dtype)
    _close(k2, *_reference(k, wk, pos, table, interleaved), dtype)


@pytest.mark.parametrize("dtype,kind", [(torch.float32, "f32"), (torch.bfloat16, "bf16")])
def test_the_fused_call_is_the_two_calls(dtype, kind):
    """Bit for bit where the pool has the source's type."""
    from zealot_amd import dense, ops
    T, H, Hkv, D = 100, 32, 8, 128
    q, k, v, (wq, wk) = _inputs(12, T, H, Hkv, D, dtype)
    table, pos = dense.rope_table(500, D), _positions(12, T, 500)
    slots = torch.randperm(10 * 16, generator=torch.Generator().manual_seed(1))[:T].cuda()
    kp, vp = _pools(10, Hkv, 16, D, kind)
    kp2, vp2 = kp.clone(), vp.clone()
    qo = ops.qk_norm_rope_append(kp, vp, q, k, v, pos, slots, table, wq, wk)
    q2, k2 = dense.qk_norm_rope(q, k, pos, table, wq, wk)
    ops.append(kp2, vp2, k2, v.contiguous(), slots)
    assert torch.equal(qo, q2) and torch.equal(kp, kp2) and torch.equal(vp, vp2)


def test_captured_and_on_another_stream():
    from zealot_amd import dense, ops
    T, H, Hkv, D = 64, 32, 8, 128
    q, k, v, (wq, wk) = _inputs(13, T, H, Hkv, D, torch.bfloat16)
    table, pos = dense.rope_table(500, D), _positions(13, T, 500)
    slots = torch.arange(T, device="cuda")
    kp, vp = _pools(6, Hkv, 16, D, "bf16")
    kp2, vp2 = kp.clone(), vp.clone()
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_append(kp2, vp2, q, k, v, pos, slots, table, wq, wk)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.qk_norm_rope_append(kp, vp, q, k, v, pos, slots, table, wq, wk, q_out=out)
    for i in range(4):
        q.normal_()
        k.normal_()
        pos.add_(1)
        g.replay()
        want = ops.qk_norm_rope_append(kp2, vp2, q, k, v, pos, slots, table, wq, wk)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kp, kp2) and torch.equal(vp, vp2), i
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = ops.qk_norm_rope_append(kp, vp, q, k, v, pos, slots, table, wq, wk, stream=s)
    s.synchronize()
    assert torch.equal(got, want)


def test_no_tokens():
    from zealot_amd import dense
    q, k, _, (wq, wk) = _inputs(14, 0, 4, 2, 64, torch.bfloat16)
    qo, ko = dense.qk_norm_rope(q, k, torch.zeros(0, dtype=torch.int32, device="cuda"), dense.rope_table(8, 64), wq, wk)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
