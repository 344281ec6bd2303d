"""Host checks of the step tables, the head norms with rotation, the page bounds,
scores and selection and the sparse decode (CPU): bad arguments are refused
before anything is launched, through the C ABI (addresses are never read) and
through the Python entry points (host tensors are refused)."""
import ctypes

import pytest
import torch

from zealot_amd import _lib, dense, ops

D = ctypes.c_void_p(0x10000)
BAD = _lib.ERR_INVALID_ARGUMENT


def _rc(rc):
    return rc, _lib.lib().zk_last_error().decode()


def _at(x):
    return ctypes.c_void_p(0x10000 + x)


def _tables(**kw):
    a = dict(bt=_at(0), n=4, mb=8, sl=_at(0x1000), nl=_at(0x2000), bs=16, nb=_at(0x3000), cnt=5, cur=_at(0x4000), end=_at(0x5000),
             slots=_at(0x6000), pos=_at(0x7000), row=_at(0x8000), rows=10, cu=_at(0x9000), kv=_at(0xa000))
    a.update(kw)
    return _rc(_lib.lib().zk_step_tables(*a.values(), None))


def test_step_tables():
    for kw in (dict(n=-1), dict(mb=0), dict(bs=0), dict(rows=-1), dict(cnt=-1), dict(mb=1 << 28, bs=16), dict(bt=None), dict(sl=None),
               dict(slots=None), dict(cu=None), dict(kv=None), dict(end=None), dict(nb=None)):
        assert _tables(**kw)[0] == BAD, kw
    for kw in (dict(kv=_at(0x1000)), dict(kv=_at(0x2008)), dict(kv=_at(0xff8)), dict(end=_at(0x4000))):  # outputs that are inputs
        rc, msg = _tables(**kw)
        assert rc == BAD and "must not be inputs" in msg, kw


def test_step_tables_outputs_apart():
    for kw in (dict(slots=_at(0)), dict(pos=_at(0x2000)), dict(row=_at(0x3010)), dict(cu=_at(0x4000)), dict(row=_at(0x7008)),
               dict(end=_at(0x9010)), dict(kv=_at(0x7c)), dict(pos=_at(0x6040)), dict(slots=_at(0xff8))):
        rc, msg = _tables(**kw)
        assert rc == BAD and "must not be inputs" in msg, kw
    assert _tables(rows=1 << 31)[0] == BAD and _tables(cnt=1 << 31)[0] == BAD


def _rope(append=False, **kw):
    T, H, Hkv, d = 10, 8, 2, 64
    row = (H + 2 * Hkv) * d
    a = dict(q=_at(0), qs=row, k=_at(2 * H * d), ks=row, v=_at(2 * (H + Hkv) * d), vs=row, dt=_lib.BF16, T=T, H=H, Hkv=Hkv, D=d, wq=None,
             wk=None, eps=1e-6, pos=_at(0x100000), rope=_at(0x200000), most=100, rot=64, inter=0, qo=_at(0x300000), qos=0)
    tail = dict(slots=_at(0x400000), bs=16, nb=10, ksc=None, vsc=None, tr=None) if append else dict(ko=_at(0x500000), kos=0)
    pools = dict(kp=_at(0x600000), vp=_at(0x700000), cd=_lib.BF16) if append else {}
    for x in (a, tail, pools):
        for key in list(kw):
            if key in x:
                x[key] = kw.pop(key)
    assert not kw
    if append:
        return _rc(_lib.lib().zk_qk_norm_rope_append(*pools.values(), *a.values(), *tail.values(), None))
    del a["v"], a["vs"]
    return _rc(_lib.lib().zk_qk_norm_rope(*a.values(), *tail.values(), None))


@pytest.mark.parametrize("append", [False, True])
def test_qk_norm_rope(append):
    for kw in (dict(dt=_lib.FP8_E4M3), dict(T=-1), dict(T=1 << 24), dict(H=0), dict(Hkv=0), dict(D=0), dict(D=1025), dict(rot=63), dict(rot=66),
               dict(rot=-2), dict(most=0), dict(q=None), dict(k=None), dict(qo=None), dict(pos=None), dict(rope=None), dict(qs=8 * 64 - 1),
               dict(ks=127), dict(qos=100), dict(H=65530)):
        rc, msg = _rope(append, **kw)
        assert rc == BAD and "zk_qk_norm_rope" in msg, kw
    assert _rope(append, T=0)[0] == _lib.OK


def test_outputs_that_overlap_other_operands():
    row = 12 * 64
    for kw in (dict(qo=_at(2)), dict(qo=_at(0), qos=row + 64), dict(qo=_at(2 * 8 * 64), qos=row), dict(ko=_at(0), kos=row),
               dict(ko=_at(0x300000)), dict(ko=_at(2 * 8 * 64), kos=row + 2), dict(qo=_at(64), qos=row)):
        rc, msg = _rope(**kw)
        assert rc == BAD and "overlaps" in msg, kw
    rc, msg = _rope(True, qo=_at(2 * 10 * 64), qos=row)
    assert rc == BAD and "overlaps" in msg


def test_qk_norm_rope_append_pools():
    for kw in (dict(kp=None), dict(vp=None), dict(cd=7), dict(bs=0), dict(nb=0), dict(slots=None), dict(v=None), dict(vs=100),
               dict(cd=_lib.FP8_E4M3), dict(ksc=D, vsc=D, tr=D)):
        assert _rope(True, **kw)[0] == BAD, kw


def test_page_bounds():
    call = lambda **kw: _rc(_lib.lib().zk_page_bounds(*dict(dict(k=D, dt=_lib.BF16, s=D, T=4, h=8, d=128, bs=16, nb=10, b=D), **kw).values(), None))  # noqa: E731
    for kw in (dict(dt=9), dict(T=-1), dict(h=0), dict(d=0), dict(bs=0), dict(nb=0), dict(k=None), dict(s=None), dict(b=None),
               dict(h=1 << 20, d=1 << 12), dict(T=1 << 40)):
        assert call(**kw)[0] == BAD, kw
    assert call(T=0, k=None, s=None, b=None)[0] == _lib.OK


def test_page_scores():
    base = dict(q=D, qd=_lib.BF16, b=D, kd=_lib.BF16, bt=D, sl=D, out=D, n=4, h=32, hkv=8, d=128, bs=16, mb=20, nb=10, mp=0)
    call = lambda **kw: _rc(_lib.lib().zk_page_scores(*dict(base, **kw).values(), None))  # noqa: E731
    for kw in (dict(qd=_lib.FP8_E4M3), dict(kd=9), dict(n=-1), dict(n=65536), dict(h=30), dict(hkv=0), dict(d=0), dict(bs=0), dict(mb=0), dict(nb=0),
               dict(mp=2), dict(q=None), dict(b=None), dict(bt=None), dict(sl=None), dict(out=None)):
        assert call(**kw)[0] == BAD, kw
    assert call(n=0, q=None)[0] == _lib.OK


def test_select_pages():
    base = dict(s=D, sl=D, n=4, hkv=8, mb=20, bs=16, k=8, sink=1, recent=1, out=D)
    call = lambda **kw: _rc(_lib.lib().zk_select_pages(*dict(base, **kw).values(), None))  # noqa: E731
    for kw in (dict(n=-1), dict(n=65536), dict(hkv=0), dict(mb=0), dict(bs=0), dict(k=0), dict(sink=-1), dict(recent=-1), dict(sink=5, recent=4),
               dict(mb=65537), dict(mb=65536, bs=1 << 16), dict(s=None), dict(sl=None), dict(out=None)):
        assert call(**kw)[0] == BAD, kw
    assert "sink" in call(k=1, sink=1, recent=1)[1]
    assert call(n=0, s=None)[0] == _lib.OK


def test_paged_decode_sparse():
    base = dict(q=D, qd=_lib.BF16, k=D, v=D, kd=_lib.BF16, o=D, bt=D, sl=D, pg=D, np=64, n=4, h=32, hkv=8, d=128, bs=16, mb=100, nb=50, sc=0.1,
                mp=0, ks=None, vs=None, ws=D, wb=1 << 30)
    call = lambda **kw: _rc(_lib.lib().zk_paged_decode_sparse(*dict(base, **kw).values(), None))  # noqa: E731
    for kw in (dict(qd=_lib.FP8_E4M3), dict(kd=9), dict(np=0), dict(n=-1), dict(n=65536), dict(h=30), dict(hkv=0), dict(d=257), dict(d=0), dict(bs=0),
               dict(mb=0), dict(nb=0), dict(h=136, hkv=8), dict(mp=5), dict(kd=_lib.FP8_E4M3), dict(ks=D, vs=D), dict(ks=D),
               dict(kd=_lib.FP8_E4M3, ks=D), dict(mb=1 << 28), dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(bt=None), dict(sl=None),
               dict(pg=None), dict(ws=None), dict(wb=16), dict(ws=_at(8)), dict(np=1 << 30)):
        assert call(**kw)[0] == BAD, kw
    assert call(n=0, q=None, ws=None)[0] == _lib.OK
    size = _lib.lib().zk_paged_decode_sparse_workspace_size
    assert size(256, 32, 8, 128, 64) == 0  # one part a list: no merge
    assert size(1, 32, 8, 128, 1024) > 0 and size(0, 32, 8, 128, 64) == 0 and size(1, 32, 8, 128, 0) == 0


def test_sizes_past_the_grids():
    lib, n = _lib.lib(), (1 << 31) - 1
    assert _rc(lib.zk_page_scores(D, _lib.BF16, D, _lib.BF16, D, D, D, 4, 32, 8, 128, 16, n, 10, 0, None))[0] == BAD
    assert _rc(lib.zk_page_scores(D, _lib.F32, D, _lib.BF16, D, D, D, 4, 32, 8, 100, 16, 1 << 26, 10, 0, None))[0] == BAD
    assert _rc(lib.zk_select_pages(D, D, 4, 8, 20, 16, n, 1, 1, D, None))[0] == BAD
    for pages in (n, 65535 * 1024 + 1):
        rc, msg = _rc(lib.zk_paged_decode_sparse(D, _lib.BF16, D, D, _lib.BF16, D, D, D, D, pages, 4, 32, 8, 128, 16, 100, 50, 0.1, 0, None,
                                                 None, D, 1 << 62, None))
        assert rc == BAD and "too many pages" in msg
        assert lib.zk_paged_decode_sparse_workspace_size(4, 32, 8, 128, pages) == 0


def test_python_entry_points_refuse_host_tensors_and_wrong_shapes():
    i32, bf = torch.int32, torch.bfloat16
    z = lambda *s, dtype=i32: torch.zeros(s, dtype=dtype)  # noqa: E731
    q, pool = z(3, 8, 64, dtype=bf), z(5, 2, 16, 64, dtype=bf)
    calls = [
        lambda: ops.step_tables(z(3, 4), z(3), z(3), 16, 10),
        lambda: ops.page_bounds(pool, z(4, dtype=torch.int64), z(5, 2, 2, 64, dtype=bf)),
        lambda: ops.page_scores(q, z(5, 2, 2, 64, dtype=bf), z(3, 4), z(3), 16),
        lambda: ops.select_pages(z(3, 2, 4, dtype=torch.float32), z(3), 16, 2),
        lambda: ops.paged_decode_sparse(q, pool, pool, z(3, 4), z(3), z(3, 2, 2)),
        lambda: dense.qk_norm_rope(q, z(3, 2, 64, dtype=bf), z(3), z(9, 64, dtype=torch.float32)),
        lambda: ops.qk_norm_rope_append(pool, pool, q, z(3, 2, 64, dtype=bf), z(3, 2, 64, dtype=bf), z(3), z(3, dtype=torch.int64),
                                        z(9, 64, dtype=torch.float32)),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError):
        ops.page_scores(q, z(5, 2, 3, 64, dtype=bf), z(3, 4), z(3), 16)
    with pytest.raises(ValueError):
        ops.step_tables(z(3), z(3), z(3), 16, 10)
    with pytest.raises(TypeError):
        ops.step_tables([1], z(3), z(3), 16, 10)
    with pytest.raises(ValueError):
        ops.select_pages(z(3, 2, 4, dtype=torch.float32), z(3), 16, 0)
    with pytest.raises(TypeError):
        dense.qk_norm_rope(z(3, 8, 64), z(3, 2, 64), z(3), None)
    for bad in ((0, 64), (8, 63), (8, 0)):
        with pytest.raises(ValueError):
            dense.rope_table(*bad, device="cpu")


def test_rope_table_on_the_host():
    t = dense.rope_table(5, 8, 100.0, device="cpu")
    assert t.shape == (5, 8) and t.dtype == torch.float32
    assert torch.equal(t[0], torch.tensor([1.0] * 4 + [0.0] * 4))
    assert abs(float(t[3, 1]) - torch.cos(torch.tensor(3 * 100.0 ** -0.25, dtype=torch.float64)).item()) <= 2.0 ** -24
