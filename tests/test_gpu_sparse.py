"""Page bounds, page scores, page selection and sparse decode on the MI355X,
each against its definition, and a run of them as a serving step makes it.

Bounds and selections are values of their inputs, so they have to be equal.
Scores: sums of 2 D products in f32, in any order and with each addition off by a
step at most: 2 D + 2 steps (2^-23) of the sum of the products' magnitudes.
Attention, with A = sum w |v| / sum w and S = the largest sum_d |q_d k_d| scale over
a row's tokens: a score (D + 4 roundings of f32) is off by e <= (D + 4) 2^-24 S, more
by 2^-8 S where an f32 query goes through bf16; a weight by a factor exp(e) and
2^-22; so numerator and denominator move the result by 2 (e + 2^-22) A, the sums by
tokens 2^-24 A each, a bf16 weight (bf16 and fp8 pools) by 2^-8 A and a bf16
output by 2^-8 of itself."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

T_OF = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}


def _randn(seed, shape, kind="f32"):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(T_OF[kind]).cuda()


def _tables(seed, lens, bs=16, slack=0):
    rng = np.random.default_rng(seed)
    pages = [-(-int(n) // bs) for n in lens]
    width = max(1, max(pages) + slack)
    perm = rng.permutation(sum(pages) + 2).astype(np.int32)
    t, o = -np.ones((len(lens), width), np.int32), 0
    for i, p in enumerate(pages):
        t[i, :p] = perm[o:o + p]
        o += p
    return torch.tensor(t).cuda(), sum(pages) + 2


def _ints(x, t=torch.int32):
    return torch.tensor(x, dtype=t, device="cuda")


# ------------------------------------------------------------------ bounds

def _same(a, b):
    """Equal values, NaN for NaN."""
    a, b = a.float().cpu(), b.float().cpu()
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    assert torch.equal(torch.nan_to_num(a, 0.0), torch.nan_to_num(b, 0.0))


def _bounds_ref(pool, slots, bounds):
    """Run after run of the slot map, token after token."""
    nb, hkv, bs, d = pool.shape
    pool, out = pool.float().cpu().numpy(), bounds.float().cpu().numpy().copy()
    slots = slots.cpu().tolist()
    last = None
    for s in slots:
        if s < 0 or s >= nb * bs:
            last = None
            continue
        b, i = divmod(s, bs)
        row = pool[b, :, i]
        if i == 0:
            out[b, :, 0] = out[b, :, 1] = row
        else:
            out[b, :, 0] = np.minimum(out[b, :, 0], row)  # (NaN stays)
            out[b, :, 1] = np.maximum(out[b, :, 1], row)
        last = s
    return torch.tensor(out)


@pytest.mark.parametrize("kind", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (2, 64, 16), (3, 96, 16), (1, 17, 16), (32, 128, 16), (2, 64, 5), (2, 32, 128)])
def test_bounds_follow_the_writes(hkv, d, bs, kind):
    """Chunks that begin and end anywhere in a page, then single tokens."""
    from zealot_amd import ops
    lens, steps = [0, 3, bs, 2 * bs + 1, 40], [[1, bs, 2 * bs + 3, 5, 0], [1, 1, 1, 1, 1], [bs - 1, 2, 1, 3 * bs, 70]]
    total = [a + sum(s[i] for s in steps) for i, a in enumerate(lens)]
    table, nb = _tables(hkv + d, total, bs)
    pool = _randn(d, (nb, hkv, bs, d), kind)
    bounds = torch.full((nb, hkv, 2, d), 7.0, device="cuda").to(T_OF[kind])
    flat = table.cpu().numpy()
    at = [0] * len(lens)
    for new in [lens] + steps:
        slots = [int(flat[i, x // bs]) * bs + x % bs for i, n in enumerate(new) for x in range(at[i], at[i] + n)]
        at = [a + n for a, n in zip(at, new)]
        slots = torch.tensor(slots + [-1, -1, nb * bs], dtype=torch.int64, device="cuda")
        want = _bounds_ref(pool, slots, bounds)
        ops.page_bounds(pool, slots, bounds)
        _same(bounds, want)


def test_bounds_of_a_large_batch_of_chunks():
    """More rows than a workgroup each: runs across the rows that one looks at."""
    from zealot_amd import ops
    rng = np.random.default_rng(1)
    new = rng.integers(1, 200, 60)
    before = rng.integers(0, 40, 60)
    table, nb = _tables(1, before + new)
    flat = table.cpu().numpy()
    slots = torch.tensor([int(flat[i, x // 16]) * 16 + x % 16 for i in range(60) for x in range(before[i], before[i] + new[i])], device="cuda")
    assert slots.numel() > 4096
    pool = _randn(2, (nb, 2, 16, 64), "bf16")
    bounds = _randn(3, (nb, 2, 2, 64), "bf16")
    want = _bounds_ref(pool, slots, bounds)
    ops.page_bounds(pool, slots, bounds)
    _same(bounds, want)


@pytest.mark.parametrize("lens", [[513], [2000, 97], [1] * 700, [300, 1, 0, 17, 16, 15, 900, 64], [4096], [4097, 3]])
def test_bounds_of_prompts_of_any_size(lens):
    """Rows past the last whole group of workgroups, runs that begin anywhere."""
    from zealot_amd import ops
    table, nb = _tables(len(lens), [n + 5 for n in lens])
    flat = table.cpu().numpy()
    slots = torch.tensor([int(flat[i, x // 16]) * 16 + x % 16 for i, n in enumerate(lens) for x in range(i % 3, n + i % 3)], device="cuda")
    pool = _randn(1, (nb, 2, 16, 64), "bf16")
    bounds = torch.stack([pool.amax(2), pool.amin(2)], 2) * 3  # of pages that begin before the run: to be extended
    want = _bounds_ref(pool, slots, bounds)
    ops.page_bounds(pool, slots, bounds)
    _same(bounds, want)


def test_bounds_of_keys_that_are_not_finite():
    from zealot_amd import ops
    pool = _randn(4, (4, 2, 16, 64), "bf16")
    pool[1, 0, 3, 5], pool[1, 1, 4, 6], pool[2, 0, 0, 0] = float("nan"), float("inf"), float("-inf")
    bounds = torch.zeros(4, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(16, 48, device="cuda")
    ops.page_bounds(pool, slots, bounds)
    _same(bounds, _bounds_ref(pool, slots, torch.zeros_like(bounds)))
    assert bool(torch.isnan(bounds[1, 0, :, 5]).all())
    ops.page_bounds(pool, torch.tensor([32 + 15], device="cuda"), bounds)  # extends what is NaN or infinite
    assert bounds[2, 0, 0, 0].item() == float("-inf")


# ------------------------------------------------------------------ scores

def _heads(H, Hkv, mapping):
    h = torch.arange(H)
    return h.view(Hkv, -1) if mapping == "grouped" else h.view(-1, Hkv).t()


def _scores_ref(q, bounds, table, lens, bs, mapping):
    q, b, table = q.double().cpu(), bounds.float().double().cpu(), table.cpu()
    N, H, D = q.shape
    nb, Hkv = b.shape[:2]
    heads = _heads(H, Hkv, mapping)
    out = torch.full((N, Hkv, table.shape[1]), -math.inf, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for n in range(N):
        for p in range(min(table.shape[1], -(-max(int(lens[n]), 0) // bs))):
            blk = int(table[n, p])
            if not 0 <= blk < nb:
                continue
            x = q[n][heads]  # [Hkv, G, D]
            t = x.clamp(max=0) * b[blk, :, None, 0] + x.clamp(min=0) * b[blk, :, None, 1]
            out[n, :, p] = t.sum(2).amax(1)
            mag[n, :, p] = (x.clamp(max=0) * b[blk, :, None, 0]).abs().add((x.clamp(min=0) * b[blk, :, None, 1]).abs()).sum(2).amax(1)
    return out, mag


SCORE_SHAPES = [(32, 8, 128, 16), (4, 4, 64, 16), (16, 8, 64, 16), (64, 8, 128, 16), (16, 1, 128, 16), (20, 4, 96, 16), (5, 1, 17, 16), (8, 2, 128, 37),
                (48, 2, 64, 16), (8, 2, 256, 16), (10, 2, 128, 16), (33, 3, 96, 16)]


@pytest.mark.parametrize("q_kind,kind", [("bf16", "bf16"), ("bf16", "fp8"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("H,Hkv,D,bs", SCORE_SHAPES)
def test_scores(H, Hkv, D, bs, q_kind, kind):
    from zealot_amd import ops
    lens = [0, 1, bs, 16 * bs, 16 * bs + 1, 70 * bs - 3, 5]
    table, nb = _tables(D, lens, bs, slack=3)
    table[5, 20], table[5, 40] = -1, nb
    q = _randn(H, (len(lens), H, D), q_kind)
    keys = torch.stack([_randn(s, (nb, Hkv, D)) for s in (1, 2)])
    bounds = torch.stack([keys.amin(0), keys.amax(0)], 2).to(T_OF[kind])
    for mapping in ("grouped", "modulo"):
        got = ops.page_scores(q, bounds, table, _ints(lens), bs, mapping=mapping).double().cpu()
        want, mag = _scores_ref(q, bounds, table, lens, bs, mapping)
        assert torch.equal(torch.isinf(got), torch.isinf(want)) and bool((got[torch.isinf(got)] < 0).all())
        fin = torch.isfinite(want)
        assert bool(((got - want).abs()[fin] <= (2 * D + 2) * 2.0 ** -23 * mag[fin] + 1e-37).all())


def test_scores_bound_the_logits():
    """Of every key in the page, in exact arithmetic; the f32 sums' error is allowed for."""
    from zealot_amd import ops
    lens = [100, 33]
    table, nb = _tables(5, lens)
    pool = _randn(6, (nb, 2, 16, 64), "bf16")
    q = _randn(7, (2, 8, 64), "bf16")
    bounds = torch.zeros(nb, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    flat = table.cpu().numpy()
    slots = torch.tensor([int(flat[i, x // 16]) * 16 + x % 16 for i, n in enumerate(lens) for x in range(n)], device="cuda")
    ops.page_bounds(pool, slots, bounds)
    s = ops.page_scores(q, bounds, table, _ints(lens), 16).double().cpu()
    for i, n in enumerate(lens):
        for x in range(n):
            k = pool[int(flat[i, x // 16]), :, x % 16].double().cpu()  # [Hkv, D]
            logits = (q[i].double().cpu().view(2, 4, 64) * k[:, None]).sum(2).amax(1)
            assert bool((s[i, :, x // 16] >= logits - 1e-3).all())


def test_scores_of_a_long_context_and_a_nan_page():
    from zealot_amd import ops
    lens = [20000, 3]
    table, nb = _tables(8, lens)
    bounds = torch.stack([-_randn(1, (nb, 8, 128)).abs(), _randn(2, (nb, 8, 128)).abs()], 2).to(torch.bfloat16)
    q = _randn(3, (2, 32, 128), "bf16")
    bounds[int(table[0, 700]), 2, 1, 9] = float("nan")
    got = ops.page_scores(q, bounds, table, _ints(lens), 16)
    assert torch.isnan(got).nonzero().tolist() == [[0, 2, 700]]
    bounds[int(table[0, 700]), 2, 1, 9] = 1.0
    want, mag = _scores_ref(q, bounds, table, lens, 16, "grouped")
    got = got.double().cpu()
    got[0, 2, 700] = want[0, 2, 700]
    fin = torch.isfinite(want)
    assert bool(((got - want).abs()[fin] <= 258 * 2.0 ** -23 * mag[fin]).all())


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("N", [60, 300])
def test_scores_of_batches(N, kind):
    """Waves of several tiles: lengths anywhere in them, blocks outside the pool."""
    from zealot_amd import ops
    Hkv, G, D, width = 8, 2, 64, 200
    rng = np.random.default_rng(N)
    lens = rng.integers(0, width * 16 + 1, N)
    lens[:5] = [0, 1, width * 16, 192 * 16, 192 * 16 + 1]
    nb = 5000
    table = _ints(rng.integers(-1, nb + 1, (N, width)))
    q = _randn(1, (N, Hkv * G, D), "f32" if kind == "f32" else "bf16")
    keys = torch.stack([_randn(s, (nb, Hkv, D)) for s in (1, 2)])
    bounds = torch.stack([keys.amin(0), keys.amax(0)], 2).to(T_OF[kind])
    got = ops.page_scores(q, bounds, table, _ints(lens), 16).double()
    ok = (table >= 0) & (table < nb) & (torch.arange(width, device="cuda") * 16 < _ints(lens)[:, None])
    b = bounds.double()[table.long().clamp(0, nb - 1)]  # [N, width, Hkv, 2, D]
    want, mag = torch.full((N, Hkv, width), -math.inf, dtype=torch.float64, device="cuda"), torch.zeros(N, Hkv, width, dtype=torch.float64, device="cuda")
    for g in range(G):
        x = q.view(N, 1, Hkv, G, D)[:, :, :, g].double()
        lo, hi = x.clamp(max=0) * b[..., 0, :], x.clamp(min=0) * b[..., 1, :]
        want = torch.maximum(want, (lo + hi).sum(-1).transpose(1, 2))
        mag = torch.maximum(mag, (lo.abs() + hi.abs()).sum(-1).transpose(1, 2))
    ok = ok[:, None].expand(N, Hkv, width)
    assert bool((got[~ok] == -math.inf).all())
    assert bool(((got - want).abs()[ok] <= (2 * D + 2) * 2.0 ** -23 * mag[ok] + 1e-37).all())


# ------------------------------------------------------------------ selection

def _select_ref(scores, lens, bs, k, sink, recent):
    x = scores.cpu().double().numpy()
    N, hkv, width = x.shape
    out = np.full((N, hkv, k), -1, np.int32)
    for n in range(N):
        held = min(width, -(-max(int(lens[n]), 0) // bs))
        for h in range(hkv):
            rank = []
            for p in range(held):
                v = x[n, h, p]
                first = 0 if p < sink or p >= held - recent else 1 if math.isnan(v) else 2
                rank.append((first, 0.0 if first < 2 else -v, p))
            best = sorted(p for _, _, p in sorted(rank)[:k])
            out[n, h, :len(best)] = best
    return torch.tensor(out)


@pytest.mark.parametrize("width", [1, 7, 64, 500, 512, 513, 2048, 2049, 8192, 8193, 33000])
@pytest.mark.parametrize("k,sink,recent", [(1, 0, 1), (1, 0, 0), (8, 2, 3), (64, 1, 2), (600, 1, 1)])
def test_selection(width, k, sink, recent):
    from zealot_amd import ops
    rng = np.random.default_rng(width + k)
    lens = [width * 16, 0, 1, max(1, width * 16 - 17), width * 8 + 3, 16 * min(width, k), 16 * min(width, k) + 1]
    x = np.round(rng.standard_normal((len(lens), 2, width)) * 4) / 4  # many equal ones
    x[0, 1] = 1.5
    scores = torch.tensor(x, dtype=torch.float32, device="cuda")
    got = ops.select_pages(scores, _ints(lens), 16, k, sink=sink, recent=recent)
    assert torch.equal(got.cpu(), _select_ref(scores, lens, 16, k, sink, recent))


def test_selection_of_values_that_are_not_finite():
    from zealot_amd import ops
    x = torch.linspace(-3, 3, 200).repeat(3, 1, 1).cuda()
    x[0, 0, 10:60:5] = float("nan")
    x[0, 0, 11] = -torch.tensor(float("nan"))
    x[1, 0, ::2] = float("-inf")
    x[1, 0, 33], x[1, 0, 35] = float("inf"), 3.4e38
    x[2, 0] = torch.where(torch.arange(200) % 2 == 0, 0.0, -0.0).cuda()  # all equal
    lens = [3200, 3190, 3185]
    for k in (1, 5, 9, 12, 120):
        got = ops.select_pages(x, _ints(lens), 16, k, sink=0, recent=1)
        assert torch.equal(got.cpu(), _select_ref(x, lens, 16, k, 0, 1)), k


def test_selection_of_the_widest_rows():
    from zealot_amd import ops
    width = 65536
    x = _randn(1, (1, 2, width))
    for n in (width * 16, 20000 * 16 + 5):
        got = ops.select_pages(x, _ints([n]), 16, 2000, sink=3, recent=3)
        assert torch.equal(got.cpu(), _select_ref(x, [n], 16, 2000, 3, 3))


# ------------------------------------------------------------------ sparse decode

def _attend_ref(q, kp, vp, table, lens, pages, mapping, ks=None, vs=None, scale=None, q_bf16=False, p_bf16=False):
    """(result, tolerance) in 64 bits, on the CPU."""
    N, H, D = q.shape
    nb, Hkv, bs, _ = kp.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    qd, kd, vd = q.double().cpu(), kp.float().double().cpu(), vp.float().double().cpu()
    table, pages = table.cpu(), pages.cpu()
    heads = _heads(H, Hkv, mapping)
    out, tol = torch.zeros(N, H, D, dtype=torch.float64), torch.zeros(N, H, D, dtype=torch.float64)
    for n in range(N):
        for h in range(Hkv):
            k, v = [], []
            for p in pages[n, h].tolist():
                if not 0 <= p < table.shape[1] or not 0 <= int(table[n, p]) < nb:
                    continue
                c = max(0, min(bs, min(int(lens[n]), table.shape[1] * bs) - p * bs))
                k.append(kd[int(table[n, p]), h, :c] * (1 if ks is None else float(ks[n, h])))
                v.append(vd[int(table[n, p]), h, :c] * (1 if vs is None else float(vs[n, h])))
            if not k or sum(len(x) for x in k) == 0:
                continue
            k, v = torch.cat(k), torch.cat(v)
            for g in heads[h].tolist():
                x = k @ qd[n, g] * scale
                w = torch.softmax(x, 0)
                out[n, g] = w @ v
                A = w @ v.abs()
                S = float((k.abs() @ qd[n, g].abs()).max()) * abs(scale)
                e = (D + 4) * 2.0 ** -24 * S + (2.0 ** -8 * S if q_bf16 else 0)
                tol[n, g] = (2 * math.expm1(e) + 2 * 2.0 ** -22 + len(x) * 2.0 ** -24 + (2.0 ** -8 if p_bf16 else 0)) * A
    return out, tol


def _lists(seed, lens, Hkv, K, bs=16):
    """Ascending random pages with the first and the last, padded with -1."""
    rng = np.random.default_rng(seed)
    out = -np.ones((len(lens), Hkv, K), np.int32)
    for n, t in enumerate(lens):
        held = -(-int(t) // bs)
        for h in range(Hkv):
            pick = rng.permutation(held)[:K]
            if held and len(pick):
                pick[0] = held - 1
            pick = np.unique(pick)
            out[n, h, :len(pick)] = pick
    return torch.tensor(out).cuda()


def _attend(q, kp, vp, table, lens, pages, mapping="grouped", ks=None, vs=None, **kw):
    from zealot_amd import ops
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), pages, mapping=mapping, k_scales=ks, v_scales=vs, **kw)
    pool, half = kp.dtype, {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}[q.dtype]
    low = pool != torch.float32
    want, tol = _attend_ref(q, kp, vp, table, lens, pages, mapping, ks, vs, kw.get("scale"), q_bf16=low and q.dtype == torch.float32, p_bf16=low)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol * (1 + half) + half * want.abs() + 1e-37).all()), float((err - tol - half * want.abs()).max())
    return got


SHAPES = [(32, 8, 128, 16), (8, 8, 128, 16), (16, 8, 64, 16), (64, 8, 128, 16), (16, 1, 64, 16), (20, 4, 96, 16), (3, 1, 40, 16), (8, 2, 256, 8),
          (8, 4, 128, 80), (8, 2, 256, 16), (10, 2, 128, 16), (64, 4, 64, 16), (26, 2, 96, 16), (17, 1, 64, 16)]


@pytest.mark.parametrize("q_kind,kind", [("bf16", "bf16"), ("bf16", "fp8"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("H,Hkv,D,bs", SHAPES)
def test_sparse_decode(H, Hkv, D, bs, q_kind, kind):
    if H // Hkv > 16:  # refused, as the decode over all pages refuses it
        from zealot_amd import ZealotError, ops
        z = torch.zeros(2, Hkv, bs, D, dtype=T_OF[kind], device="cuda")
        with pytest.raises(ZealotError):
            ops.paged_decode_sparse(_randn(1, (1, H, D), q_kind), z, z, _ints([[0]]), _ints([1]), _ints([[[0]] * Hkv]),
                                    k_scales=None if kind != "fp8" else torch.ones(1, Hkv, device="cuda"),
                                    v_scales=None if kind != "fp8" else torch.ones(1, Hkv, device="cuda"))
        return
    lens = [0, 1, bs, bs + 1, 5 * bs - 1, 40 * bs + 3]
    table, nb = _tables(H + D, lens, bs, slack=2)
    kp, vp, q = _randn(1, (nb, Hkv, bs, D), kind), _randn(2, (nb, Hkv, bs, D), kind), _randn(3, (len(lens), H, D), q_kind)
    ks, vs = [(0.5 + torch.rand(len(lens), Hkv, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (4, 5)]
    for mapping in ("grouped", "modulo"):
        for K in (1, 9, 33):
            got = _attend(q, kp, vp, table, lens, _lists(K, lens, Hkv, K, bs), mapping, ks, vs)
            assert bool((got[0] == 0).all())


@pytest.mark.parametrize("kind,D,G", [("bf16", 128, 4), ("fp8", 128, 4), ("f32", 128, 4), ("bf16", 64, 1), ("fp8", 64, 8)])
@pytest.mark.parametrize("N,K", [(1, 1100), (1, 300), (3, 130), (40, 64), (70, 48)])
def test_long_lists_and_batches(N, K, kind, D, G):
    """Lists in parts with a merge, and batches of one part a list."""
    rng = np.random.default_rng(N + K)
    lens = rng.integers(1, K * 16 + 200, N).tolist()
    lens[0] = K * 16 + 100
    table, nb = _tables(N, lens)
    Hkv = 2
    kp, vp, q = _randn(1, (nb, Hkv, 16, D), kind), _randn(2, (nb, Hkv, 16, D), kind), _randn(3, (N, Hkv * G, D), "f32" if kind == "f32" else "bf16")
    ks, vs = [(0.5 + torch.rand(N, Hkv, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (4, 5)]
    _attend(q, kp, vp, table, lens, _lists(K, lens, Hkv, K), "grouped", ks, vs)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("fp8", 64), ("f32", 128), ("bf16", 96)])
def test_lists_of_any_kind(kind, D):
    """Descending lists, repeated pages, holes, pages behind the length or the
    table, blocks outside the pool, lists without a page."""
    lens = [100, 100, 100, 100, 100, 33]
    table, nb = _tables(9, lens, slack=3)
    table[3, 2], table[3, 4] = -1, nb + 5
    lists = [[6, 5, 3, 0, 1, 2], [6, 6, 2, 2, 2, -1], [-1, 4, -1, -1, 6, -1], [0, 1, 2, 3, 4, 5], [-1] * 6, [9, 2, 200, -7, 2 ** 31 - 1, 1]]
    pages = _ints([[x, x[::-1]] for x in lists])
    kp, vp, q = _randn(1, (nb, 2, 16, D), kind), _randn(2, (nb, 2, 16, D), kind), _randn(3, (6, 8, D), "f32" if kind == "f32" else "bf16")
    ks, vs = [(0.5 + torch.rand(6, 2, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (4, 5)]
    got = _attend(q, kp, vp, table, lens, pages, "grouped", ks, vs)
    assert bool((got[4] == 0).all())


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f32", 128), ("bf16", 96)])
def test_what_lies_behind_the_length_does_not_count(kind, D):
    lens = [37, 5, 16]
    table, nb = _tables(10, lens)
    kp, vp, q = _randn(1, (nb, 2, 16, D), kind), _randn(2, (nb, 2, 16, D), kind), _randn(3, (3, 8, D), "f32" if kind == "f32" else "bf16")
    pages = _lists(1, lens, 2, 4)
    want = _attend(q, kp, vp, table, lens, pages)
    for i, n in enumerate(lens):
        if n % 16:
            kp[int(table[i, n // 16]), :, n % 16:], vp[int(table[i, n // 16]), :, n % 16:] = float("nan"), float("inf")
    from zealot_amd import ops
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), pages)
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f32", 128), ("bf16", 96)])
def test_scores_of_minus_infinity_and_nan(kind, D):
    """Keys whose scores are -inf have weight 0; a row of nothing else, or with a NaN, is NaN, in its own sequence only."""
    from zealot_amd import ops
    lens = [40, 40, 40]
    table, nb = _tables(11, lens)
    kp, vp, q = _randn(1, (nb, 1, 16, D), kind), _randn(2, (nb, 1, 16, D), kind), _randn(3, (3, 4, D), "f32" if kind == "f32" else "bf16").abs()
    kp[int(table[0, 0]), 0, 3] = float("-inf")
    for p in range(3):
        kp[int(table[1, p]), 0] = float("-inf")
    kp[int(table[2, 1]), 0, 7, 1] = float("nan")
    pages = _ints([[[0, 1, 2]]] * 3)
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), pages)
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
    k = kp[table[0].long(), 0].flatten(0, 1)[:40].double().cpu()
    v = vp[table[0].long(), 0].flatten(0, 1)[:40].double().cpu()
    x = (q[0].double().cpu() @ k.t()) / math.sqrt(D)
    want = torch.softmax(x, 1) @ v
    assert float((got[0].double().cpu() - want).abs().max()) <= 2.0 ** -7 * float(v.abs().max())


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f32", 128), ("bf16", 96)])
def test_values_of_infinity_stay_infinite(kind, D):
    """Every weight is positive here (scores within a few units), 1 exactly in the first two rows."""
    from zealot_amd import ops
    lens = [1, 40, 40]
    table, nb = _tables(13, lens)
    kp, vp, q = _randn(1, (nb, 1, 16, D), kind), _randn(2, (nb, 1, 16, D), kind), _randn(3, (3, 4, D), "f32" if kind == "f32" else "bf16")
    for p in range(3):
        kp[int(table[1, p]), 0] = 0
    for i in range(3):
        vp[int(table[i, 0]), 0, 0, 3], vp[int(table[i, 0]), 0, 0, 6] = float("inf"), float("-inf")
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), _ints([[[0, 1, 2]]] * 3)).float().cpu()
    assert bool((got[:, :, 3] == float("inf")).all()) and bool((got[:, :, 6] == float("-inf")).all())
    rest = [d for d in range(D) if d not in (3, 6)]
    assert bool(torch.isfinite(got[:, :, rest]).all())
    assert torch.equal(got[0, :, rest], vp[int(table[0, 0]), 0, 0].float().cpu()[rest].expand(4, -1))


def test_all_pages_are_the_dense_decode():
    from zealot_amd import ops
    lens = [100, 1, 700, 64]
    table, nb = _tables(12, lens)
    kp, vp, q = _randn(1, (nb, 8, 16, 128), "bf16"), _randn(2, (nb, 8, 16, 128), "bf16"), _randn(3, (4, 32, 128), "bf16")
    width = table.shape[1]
    pages = torch.arange(width, dtype=torch.int32, device="cuda").expand(4, 8, width).contiguous()
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), pages).float()
    want = ops.paged_decode(q, kp, vp, table, _ints(lens)).float()
    A = float(vp.float().abs().max())
    assert float((got - want).abs().max()) <= 2 * 2.0 ** -8 * 2 * A  # each within a weight's and an output's rounding


def test_scale_and_given_outputs():
    from zealot_amd import ops
    lens = [500]
    table, nb = _tables(13, lens)
    kp, vp, q = _randn(1, (nb, 2, 16, 64), "bf16"), _randn(2, (nb, 2, 16, 64), "bf16"), _randn(3, (1, 8, 64), "bf16")
    pages = _lists(2, lens, 2, 20)
    out = torch.empty_like(q)
    ws = torch.empty(ops.sparse_workspace_bytes(1, 8, 2, 64, 20), dtype=torch.uint8, device="cuda")
    got = _attend(q, kp, vp, table, lens, pages, scale=0.03, out=out, workspace=ws)
    assert got is out


def test_a_step_from_lengths_to_attention():
    """Tables and slots from lengths, norm, rotation and write, bounds, scores,
    selection and attention, step after step, eagerly and as a replayed graph;
    each step's result against attention over the same pages in 64 bits, and
    with every page selected against the dense decode."""
    from zealot_amd import dense, ops
    N, H, Hkv, D, bs, K = 6, 8, 2, 64, 16, 4
    lens = _ints([0] * N)
    table = torch.full((N, 12), -1, dtype=torch.int32, device="cuda")
    nb = 80
    blocks = torch.randperm(nb, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    cursor = torch.zeros(1, dtype=torch.int64, device="cuda")
    kp, vp = torch.zeros(nb, Hkv, bs, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(nb, Hkv, bs, D, dtype=torch.bfloat16, device="cuda")
    bounds = torch.zeros(nb, Hkv, 2, D, dtype=torch.bfloat16, device="cuda")
    rope = dense.rope_table(256, D)
    wq, wk = [1 + 0.1 * _randn(s, (D,)) for s in (1, 2)]
    wq, wk = wq.bfloat16(), wk.bfloat16()

    def write(new, rows, x, out=None):
        t = ops.step_tables(table, lens, new, bs, rows, blocks, cursor, out=out)
        q, k, v = [y.unflatten(1, (-1, D)) for y in x.split((H * D, Hkv * D, Hkv * D), 1)]
        q = ops.qk_norm_rope_append(kp, vp, q, k, v, t.positions, t.slot_mapping, rope, wq, wk)
        ops.page_bounds(kp, t.slot_mapping, bounds)
        return t, q

    def attend(t, q):
        s = ops.page_scores(q, bounds, table, t.kv_lens, bs)
        pages = ops.select_pages(s, t.kv_lens, bs, K)
        return pages, ops.paged_decode_sparse(q, kp, vp, table, t.kv_lens, pages)

    prompt = [30, 1, 16, 100, 0, 64]
    t, _ = write(_ints(prompt), sum(prompt) + 3, _randn(5, (sum(prompt) + 3, (H + 2 * Hkv) * D), "bf16"))
    lens.copy_(t.kv_lens)
    cursor.copy_(t.cursor)
    one = torch.ones(N, dtype=torch.int32, device="cuda")
    x = _randn(6, (N, (H + 2 * Hkv) * D), "bf16")

    def check(t, q, pages, got):
        n = t.kv_lens.cpu().tolist()
        want, tol = _attend_ref(q, kp, vp, table, n, pages, "grouped", p_bf16=True)
        assert bool(((got.double().cpu() - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all())
        every = torch.arange(12, dtype=torch.int32, device="cuda").expand(N, Hkv, 12).contiguous()
        a = ops.paged_decode_sparse(q, kp, vp, table, t.kv_lens, every).float()
        b = ops.paged_decode(q, kp, vp, table, t.kv_lens).float()
        assert float((a - b).abs().max()) <= 2.0 ** -6 * float(vp.float().abs().max())

    for step in range(3):
        x.copy_(_randn(10 + step, x.shape, "bf16"))
        t, q = write(one, N, x)
        pages, got = attend(t, q)
        check(t, q, pages, got)
        lens.copy_(t.kv_lens)
        cursor.copy_(t.cursor)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, q = write(one, N, x)
        pages, got = attend(t, q)
    for step in range(20):  # past a block's end of every sequence
        x.copy_(_randn(20 + step, x.shape, "bf16"))
        g.replay()
        torch.cuda.synchronize()
        check(t, q, pages, got)
        p2, g2 = attend(t, q)
        assert torch.equal(p2, pages) and torch.equal(g2, got)
        lens.copy_(t.kv_lens)
        cursor.copy_(t.cursor)
    assert int(cursor) <= nb


def test_another_stream_and_two_at_once():
    from zealot_amd import ops
    lens = [3000, 2000]
    table, nb = _tables(14, lens)
    kp, vp, q = _randn(1, (nb, 2, 16, 128), "bf16"), _randn(2, (nb, 2, 16, 128), "bf16"), _randn(3, (2, 8, 128), "bf16")
    pages = _lists(3, lens, 2, 64)
    n = _ints(lens)
    want = ops.paged_decode_sparse(q, kp, vp, table, n, pages)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [ops.paged_decode_sparse(q, kp, vp, table, n, pages, stream=s) for _ in range(5) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("D", [128, 80])
def test_pools_past_32_bits(D):
    """The same step on a small pool and on one whose last blocks lie more than 2^32 elements in: equal results."""
    from zealot_amd import dense, ops
    H, Hkv, bs, small = 32, 8, 16, 40
    nb = 2 ** 32 // (Hkv * bs * D) + 100
    lens = [200, 33, 290]
    table, used = _tables(21, lens)
    assert used <= small
    x = _randn(22, (sum(lens), (H + 2 * Hkv) * D), "bf16")
    q, k, v = [y.unflatten(1, (-1, D)) for y in x.split((H * D, Hkv * D, Hkv * D), 1)]
    rope, qd, results = dense.rope_table(300, D), _randn(23, (3, H, D), "bf16"), []
    for blocks in (small, nb):
        far = torch.where((table >= 0) & (table % 2 == 0), table + blocks - small, table)
        kp, vp = [torch.empty(blocks, Hkv, bs, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        bounds = torch.empty(blocks, Hkv, 2, D, dtype=torch.bfloat16, device="cuda")
        t = ops.step_tables(far, _ints([0] * 3), _ints(lens), bs, sum(lens))
        qo = ops.qk_norm_rope_append(kp, vp, q, k, v, t.positions, t.slot_mapping, rope)
        ops.page_bounds(kp, t.slot_mapping, bounds)
        s = ops.page_scores(qd, bounds, far, t.kv_lens, bs)
        pages = ops.select_pages(s, t.kv_lens, bs, 6)
        results.append((qo, s, pages, ops.paged_decode_sparse(qd, kp, vp, far, t.kv_lens, pages)))
        assert blocks == small or int(t.slot_mapping.max()) * Hkv * D > 2 ** 32 - 2 ** 24
        del kp, vp, bounds
    torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def _off(x):
    """A copy of x whose first element lies one element behind an aligned address."""
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
    return y.copy_(x)


@pytest.mark.parametrize("kind", ["f32", "bf16", "fp8"])
def test_operands_off_their_alignment(kind):
    from zealot_amd import ops
    lens = [100, 1, 700, 64]
    table, nb = _tables(15, lens)
    kp, vp, q = [_off(_randn(s, sh, t)) for s, sh, t in ((1, (nb, 2, 16, 128), kind), (2, (nb, 2, 16, 128), kind), (3, (4, 8, 128), "bf16"))]
    ks, vs = [(0.5 + torch.rand(4, 2, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (4, 5)]
    _attend(q, kp, vp, table, lens, _lists(1, lens, 2, 9), "grouped", ks, vs, out=_off(torch.zeros(4, 8, 128, dtype=torch.bfloat16)))
    slots = torch.cat([table[i].repeat_interleave(16).long()[:n] * 16 + torch.arange(n, device="cuda") % 16 for i, n in enumerate(lens)])
    bounds = _off(torch.zeros(nb, 2, 2, 128, dtype=T_OF[kind], device="cuda"))
    want = _bounds_ref(kp, slots, bounds)
    ops.page_bounds(kp, slots, bounds)
    _same(bounds, want)
    got = ops.page_scores(q, bounds, table, _ints(lens), 16).double().cpu()
    want, mag = _scores_ref(q, bounds, table, lens, 16, "grouped")
    fin = torch.isfinite(want)
    assert torch.equal(torch.isinf(got), ~fin) and bool(((got - want).abs()[fin] <= 258 * 2.0 ** -23 * mag[fin] + 1e-37).all())


def test_two_graphs_over_one_workspace():
    """Parts of a list are written before they are read within each call, so graphs that run in turn may share it."""
    from zealot_amd import ops
    sets = []
    for seed, lens in ((30, [3000, 2000]), (31, [900, 5000])):
        table, nb = _tables(seed, lens)
        sets.append((_randn(seed, (2, 8, 128), "bf16"), _randn(1, (nb, 2, 16, 128), "bf16"), _randn(2, (nb, 2, 16, 128), "bf16"), table, _ints(lens),
                     _lists(seed, lens, 2, 64)))
    ws = torch.empty(ops.sparse_workspace_bytes(2, 8, 2, 128, 64), dtype=torch.uint8, device="cuda")
    want = [ops.paged_decode_sparse(*s) for s in sets]
    outs, graphs = [torch.empty_like(w) for w in want], []
    torch.cuda.synchronize()
    for s, out in zip(sets, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_decode_sparse(*s, out=out, workspace=ws)
        graphs.append(g)
    for _ in range(4):
        for g, out, w in zip(graphs, outs, want):
            out.zero_()
            g.replay()
            ws.add_(1)
            torch.cuda.synchronize()
            assert torch.equal(out, w)
