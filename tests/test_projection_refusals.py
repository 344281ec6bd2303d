"""Host checks of the 8-bit projections and of the low-rank adapters (CPU): bad
arguments are refused before anything is launched, through the C ABI (addresses
are never read) and through the Python entry points (host tensors are refused)."""
import ctypes

import pytest
import torch

from zealot_amd import _lib, dense

BAD, OK = _lib.ERR_INVALID_ARGUMENT, _lib.OK
I64 = ctypes.c_int64


def _at(x):
    return ctypes.c_void_p(0x10000000 + x)


def _rc(rc):
    return rc, _lib.lib().zk_last_error().decode()


def _norm(**kw):
    a = dict(x=_at(0), r=_at(0x100000), w=_at(0x200000), q=_at(0x300000), s=_at(0x400000), ro=_at(0x500000), rows=None, xr=10, n=10, dim=256,
             eps=1e-6, dt=_lib.BF16)
    a.update(kw)
    return _rc(_lib.lib().zk_rms_norm_fp8(*a.values(), None))


def test_rms_norm_fp8():
    for kw in (dict(dt=_lib.FP8_E4M3), dict(n=-1, xr=-1), dict(dim=0), dict(dim=32769), dict(n=1 << 31, xr=1 << 31), dict(n=9), dict(x=None), dict(w=None),
               dict(q=None), dict(s=None), dict(ro=None), dict(rows=_at(0x600000), xr=-1)):
        rc, msg = _norm(**kw)
        assert rc == BAD and "zk_rms_norm_fp8" in msg, kw
    assert _norm(n=0, xr=0, x=None, q=None)[0] == OK
    assert _norm(n=0, rows=_at(0x600000))[0] == OK
    # rows that do not fit a workgroup's registers: element by element past 4096, f32 past 16384
    assert "too long" in _norm(dim=4097, xr=1, n=1)[1]
    assert "too long" in _norm(dim=16388, xr=1, n=1, dt=_lib.F32, r=None)[1]


def test_rms_norm_fp8_overlaps():
    for kw in (dict(q=_at(16)), dict(q=_at(0x100000)), dict(s=_at(0x200010)), dict(ro=_at(0x100002)), dict(ro=_at(0x200000)), dict(ro=_at(2)),
               dict(ro=_at(0x300010)), dict(s=_at(0x300000)), dict(rows=_at(0x300000)),
               dict(rows=_at(0x600000), ro=_at(0)), dict(rows=_at(0x600000), ro=_at(0x100000))):  # (in place: all rows, or another reads them)
        rc, msg = _norm(**kw)
        assert rc == BAD and "overlap" in msg, kw


def test_silu_mul_fp8():
    base = dict(g=_at(0), u=_at(512), q=_at(0x300000), s=_at(0x400000), rows=10, cols=256, gs=512, us=512, dt=_lib.BF16)
    call = lambda **kw: _rc(_lib.lib().zk_silu_mul_fp8(*dict(base, **kw).values(), None))  # noqa: E731
    for kw in (dict(dt=_lib.FP8_E4M3), dict(rows=-1), dict(cols=0), dict(cols=32769, gs=0, us=0), dict(gs=255), dict(us=100), dict(us=1 << 32), dict(g=None),
               dict(u=None), dict(q=None), dict(s=None), dict(q=_at(1000)), dict(s=_at(0)), dict(s=_at(0x300004)), dict(q=_at(512 * 19)),
               dict(cols=4097, gs=0, us=0)):
        assert call(**kw)[0] == BAD, kw
    assert call(rows=0, g=None)[0] == OK


def test_fp8_weight():
    size = _lib.lib().zk_fp8_weight_bytes
    assert size(64, 128) == 8192 and size(1, 1) == 8192 and size(65, 129) == 4 * 8192
    assert size(0, 1) == 0 and size(1, 0) == 0 and size((1 << 22) + 1, 1) == 0
    base = dict(w=_at(0), dt=_lib.BF16, p=_at(0x300000), s=_at(0x500000), n=100, k=300)
    call = lambda **kw: _rc(_lib.lib().zk_fp8_weight(*dict(base, **kw).values(), None))  # noqa: E731
    for kw in (dict(dt=7), dict(n=0), dict(k=0), dict(n=(1 << 22) + 1), dict(w=None), dict(p=None), dict(s=None), dict(p=_at(8)), dict(p=_at(0x300008)),
               dict(p=_at(1024)), dict(s=_at(100)), dict(s=_at(0x300100))):
        assert call(**kw)[0] == BAD, kw


def test_linear_fp8():
    base = dict(x=_at(0), xs=_at(0x100000), w=_at(0x200000), ws=_at(0x300000), y=_at(0x400000), m=10, n=100, k=256, dt=_lib.BF16, wk=None, wb=0)
    call = lambda **kw: _rc(_lib.lib().zk_linear_fp8(*dict(base, **kw).values(), None))  # noqa: E731
    for kw in (dict(dt=_lib.FP8_E4M3), dict(m=-1), dict(n=0), dict(k=0), dict(k=250), dict(k=8), dict(m=1 << 25), dict(n=1 << 25), dict(k=1 << 25),
               dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(x=_at(8)), dict(w=_at(0x200008)), dict(y=_at(0x400004)),
               dict(y=_at(0)), dict(y=_at(0x100000)), dict(y=_at(0x200100)), dict(y=_at(0x300000)), dict(m=1 << 24, n=1 << 22)):
        rc, msg = call(**kw)
        assert rc == BAD and "zk_linear_fp8" in msg, kw
    assert call(m=0, x=None)[0] == OK
    # k split over workgroups: the sums need room
    far = dict(m=64, n=4096, k=14336, x=_at(0), xs=_at(0x1000000), w=_at(0x2000000), ws=_at(0x9000000), y=_at(0xa000000), wk=_at(0xb000000), wb=1 << 26)
    size = _lib.lib().zk_linear_fp8_workspace_size(64, 4096, 14336, _lib.BF16)
    assert size > 0 and _lib.lib().zk_linear_fp8_workspace_size(16, 4096, 14336, _lib.BF16) == 0
    assert _lib.lib().zk_linear_fp8_workspace_size(0, 4096, 14336, _lib.BF16) == 0 and _lib.lib().zk_linear_fp8_workspace_size(64, 4096, 14330, _lib.BF16) == 0
    for kw in (dict(wk=None), dict(wb=size - 1), dict(wk=_at(0xb000008)), dict(wk=_at(0x2000000)), dict(wk=_at(0xa000000)), dict(wk=_at(0x1000000 - 16))):
        rc, msg = call(**dict(far, **kw))
        assert rc == BAD and "zk_linear_fp8" in msg, kw


def _plan(**kw):
    a = dict(ids=_at(0), n=100, na=7, order=_at(0x1000), off=_at(0x2000), tiles=_at(0x3000))
    a.update(kw)
    return _rc(_lib.lib().zk_lora_plan(*a.values(), None))


def test_lora_plan():
    for kw in (dict(n=-1), dict(n=(1 << 24) + 1), dict(na=0), dict(na=2049), dict(ids=None), dict(order=None), dict(off=None), dict(tiles=None),
               dict(tiles=_at(0x3004)), dict(order=_at(0x10)), dict(off=_at(0x1004)), dict(tiles=_at(0x1000)), dict(off=_at(0x3008))):
        rc, msg = _plan(**kw)
        assert rc == BAD and "zk_lora_plan" in msg, kw
    tiles = _lib.lib().zk_lora_max_tiles
    assert tiles(100, 7) == 6 + 7 and tiles(3, 100) == 3 and tiles(0, 5) == 0 and tiles(5, 0) == 0 and tiles(5, 2049) == 0


def _lora(**kw):
    a = dict(x=_at(0), xsc=None, xst=0, xd=_lib.BF16, a=_at(0x1000000), b=_at(0x2000000), sc=_at(0x3000000), dt=_lib.BF16, order=_at(0x3100000),
             tiles=_at(0x3300000), n=50, na=4, k=256, cols=192, rank=16, parts=1, pc=None, pb=0, y=_at(0x4000000), ys=0,
             ws=_at(0x5000000), wb=1 << 24)
    a.update(kw)
    return _rc(_lib.lib().zk_lora(*a.values(), None))


def test_lora():
    for kw in (dict(dt=_lib.FP8_E4M3, xd=_lib.FP8_E4M3), dict(xd=_lib.F32), dict(dt=_lib.F32, xd=_lib.FP8_E4M3, xsc=_at(0x3400000)), dict(xd=_lib.FP8_E4M3),
               dict(xsc=_at(0x3400000)), dict(n=-1), dict(n=(1 << 24) + 1), dict(na=0), dict(na=2049), dict(k=0), dict(cols=0), dict(rank=0), dict(rank=257),
               dict(parts=0), dict(parts=5), dict(parts=3, rank=171, pc=(I64 * 3)(64, 64, 64)), dict(parts=2), dict(parts=2, pc=(I64 * 2)(100, 93)),
               dict(parts=2, pc=(I64 * 2)(192, 0)), dict(parts=2, pc=(I64 * 2)(-10, 202)), dict(parts=2, pc=(I64 * 2)(1 << 40, 1 << 40)), dict(pb=-1),
               dict(parts=2, pb=64), dict(xst=255), dict(ys=100), dict(x=None), dict(a=None), dict(b=None), dict(order=None),
               dict(tiles=None), dict(y=None), dict(ws=None), dict(wb=100), dict(ws=_at(0x5000008)), dict(tiles=_at(0x3300004)), dict(cols=1 << 24),
               dict(k=1 << 24)):
        rc, msg = _lora(**kw)
        assert rc == BAD and "zk_lora" in msg, kw
    for kw in (dict(y=_at(0x100)), dict(y=_at(0x1000000)), dict(y=_at(0x2000000)), dict(y=_at(0x3000000)), dict(y=_at(0x3100000)), dict(ws=_at(0)),
               dict(ws=_at(0x2000000)), dict(ws=_at(0x4000000)), dict(ws=_at(0x3300000))):
        rc, msg = _lora(**kw)
        assert rc == BAD and "overlaps" in msg, kw
    assert _lora(n=0, x=None, y=None, ws=None)[0] == OK
    size = _lib.lib().zk_lora_workspace_size
    assert size(50, 4, 256, 16, 1, _lib.BF16) >= 50 * 16 * 4 and size(0, 4, 256, 16, 1, _lib.BF16) == 0 and size(50, 4, 256, 300, 1, _lib.BF16) == 0


def test_python_entry_points_refuse_host_tensors_and_wrong_shapes():
    bf, f8 = torch.bfloat16, torch.float8_e4m3fn
    z = lambda *s, dtype=bf: torch.zeros(s, dtype=dtype)  # noqa: E731
    rows = dense.Fp8Rows(torch.zeros((3, 128), dtype=torch.uint8).view(f8), z(3, dtype=torch.float32))
    weight = dense.Fp8Weight(torch.zeros(8192, dtype=torch.uint8), z(64, dtype=torch.float32), 64, 128)
    plan = dense.LoraPlan(z(3, dtype=torch.int32), z(3, dtype=torch.int32), z(2, 2, dtype=torch.int32))
    calls = [lambda: dense.rms_norm_fp8(z(3, 64), z(64)), lambda: dense.silu_mul_fp8(z(3, 64), z(3, 64)), lambda: dense.fp8_weight(z(64, 128)),
             lambda: dense.linear_fp8(rows, weight), lambda: dense.lora_plan(z(3, dtype=torch.int32), 2),
             lambda: dense.lora(z(3, 64), z(2, 16, 64), z(2, 32, 16), None, plan, z(3, 32))]
    for call in calls:
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        dense.rms_norm_fp8(z(3, 64, dtype=torch.float16), z(64))
    with pytest.raises(ValueError):
        dense.rms_norm_fp8(z(3, 4, 16), z(16))
    with pytest.raises(TypeError):
        dense.linear_fp8(rows, z(64, 128))
    with pytest.raises(ValueError):
        dense.linear_fp8(dense.Fp8Rows(rows.data[:, :64], rows.scales), weight)
    with pytest.raises(ValueError):
        dense.Fp8Weight(torch.zeros(8000, dtype=torch.uint8), z(64, dtype=torch.float32), 64, 128)
    with pytest.raises(ValueError):
        dense.Fp8Weight(torch.zeros(8192, dtype=torch.uint8), z(63, dtype=torch.float32), 64, 128)
    with pytest.raises(ValueError):
        dense.fp8_weight(z(64, 128), z(64, dtype=torch.float32))
    with pytest.raises(ValueError):
        dense.fp8_weight(torch.zeros((64, 128), dtype=torch.uint8).view(f8))
    with pytest.raises(ValueError):
        dense.lora_plan(z(3, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="add up"):
        dense.lora(z(3, 64), z(2, 32, 64), z(2, 32, 16), None, plan, z(3, 32), parts=(16, 17))
    with pytest.raises(ValueError):
        dense.lora(z(3, 64), z(2, 32, 64), z(2, 32, 16), None, plan, z(3, 32), parts=(16, 16), part_block=16)


def test_rowmajor_of_a_packed_weight_on_the_host():
    """The packed order as the header states it, byte by byte."""
    n, k = 70, 200
    p = torch.zeros(2 * 4 * 2 * 2048, dtype=torch.uint8)
    w = torch.randint(0, 120, (n, k), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    for r in range(n):
        G, i1, t, i0 = r // 64, r % 64 // 16, r % 16 // 4, r % 4
        for c in range(k):
            p[(((G * 4 + t) * 2 + c // 128) * 8 + c % 128 // 16) * 256 + (4 * i1 + i0) * 16 + c % 16] = w[r, c]
    got = dense.Fp8Weight(p, torch.ones(n), n, k).rowmajor()
    assert torch.equal(got.view(torch.uint8), w)
