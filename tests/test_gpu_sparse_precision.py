"""Digits of the sparse decode: f32 queries on every pool, weights, and the decode over all pages.

Tolerances, in shares of A = sum w |v| of an element, u = 2^-24, S the largest
sum |q_d k_d| * scale of its row, n its tokens:
  scores    a sum of `parts` D rounded additions, then the two products with the
            scale, log2 e and a key scale and the difference from the maximum:
            e = (parts D + 4) u S, which moves a weight by expm1(e), in the sum over
            the values and in the sum of the weights: 2 expm1(e)
  exp2      2^-22 a weight, twice; the rescaling of the waves' and the parts' results
            2^-22 each, twice
  sums      3 n u over the values (weights in up to three parts), n u over the weights, 3 u behind
  weights   bf16 queries on bf16 and fp8 pools: their leading 8 bits cut (what is left is below 2^-7
            of the weight), the rest rounded to 8 bits: 2^-7 2^-8 = 2^-15; 2^-20 is added.  f32 queries:
            their 24 bits, up to 2^-29 where parts would be zero
and half a step of a bf16 output, 2^-8 of the value."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
T_OF = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def attend64(q, k, v, scale):
    """(sum w v, sum w |v|, S) of one head row q [D] over k, v [n, D] in 64 bits."""
    x = k @ q * scale
    w = torch.softmax(x, 0)
    return w @ v, w @ v.abs(), float((k.abs() @ q.abs()).max()) * scale


def tolerance(A, S, n, D, parts=1, low=True):
    e = (parts * D + 4) * U * S
    return A * (2 * math.expm1(e) + 4 * 2.0 ** -22 + (4 * n + 3) * U + (2.0 ** -15 + 2.0 ** -20 if low else 2.0 ** -29)) * (1 + 2.0 ** -10)


def between(shape, seed):
    """f32 values between two bf16 ones, all above the nearer one: rounded to 8 bits, a sum of them is off one way."""
    g = torch.Generator().manual_seed(seed)
    x = 0.5 + torch.rand(shape, generator=g)
    x = x.bfloat16().float()
    return x + torch.exp2(torch.floor(torch.log2(x))) * 2.0 ** -7 * 0.44


def rows_of(seed, n, D, kind):
    """Keys whose scores with positive queries spread from one sign to the other, and values."""
    g = torch.Generator().manual_seed(seed)
    c = torch.linspace(-1, 1, n)[torch.randperm(n, generator=g)]
    k = c[:, None] * (0.75 + 0.5 * torch.rand(n, D, generator=g))
    return k.to(T_OF[kind]), torch.randn(n, D, generator=g).to(T_OF[kind])


def problem(seed, lens, H, Hkv, D, kind, bs):
    """Pools of shuffled blocks, each sequence's rows in them: (kp, vp, table, keys, values)."""
    pages = [-(-n // bs) for n in lens]
    nb = sum(pages) + 2
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
    table = -torch.ones(len(lens), max(pages), dtype=torch.int32)
    kp, vp = torch.zeros(nb, Hkv, bs, D), torch.zeros(nb, Hkv, bs, D)
    keys, values, at = [], [], 0
    for i, n in enumerate(lens):
        both = [rows_of(seed + 100 * i + h, n, D, kind) for h in range(Hkv)]
        keys.append([k.double() if kind != "fp8" else k.float().double() for k, _ in both])
        values.append([v.double() if kind != "fp8" else v.float().double() for _, v in both])
        for p in range(pages[i]):
            b, c = order[at], min(bs, n - p * bs)
            at += 1
            table[i, p] = b
            for h in range(Hkv):
                kp[b, h, :c] = keys[i][h][p * bs:p * bs + c].float()
                vp[b, h, :c] = values[i][h][p * bs:p * bs + c].float()
    return kp.to(T_OF[kind]).cuda(), vp.to(T_OF[kind]).cuda(), table.cuda(), keys, values


def every_page(table, Hkv):
    n, width = table.shape
    return torch.arange(width, dtype=torch.int32, device="cuda").expand(n, Hkv, width).contiguous()


def check(got, q, keys, values, Hkv, scale, parts, low, ks=None, vs=None, half=0.0):
    N, H, D = q.shape
    G = H // Hkv
    for i in range(N):
        for j in range(H):
            h = j // G
            k, v = keys[i][h], values[i][h]
            if ks is not None:
                k, v = k * float(ks[i, h]), v * float(vs[i, h])
            want, A, S = attend64(q[i, j].double().cpu(), k, v, scale)
            err = (got[i, j].double().cpu() - want).abs()
            tol = tolerance(A, S, len(k), D, parts, low)
            assert bool((err <= tol * (1 + half) + half * want.abs()).all()), (i, j, float((err / tol).max()))


def test_a_query_rounded_to_8_bits_is_outside_the_tolerance():
    """What the check below is worth, on the CPU: such queries rounded to bf16 miss it by far."""
    for D in (64, 96, 128, 256):
        q = between((D,), D)
        k, v = [x.double() for x in rows_of(D, 40, D, "bf16")]
        scale = 2.0 / D
        want, A, S = attend64(q.double(), k, v, scale)
        low, _, _ = attend64(q.bfloat16().double(), k, v, scale)
        assert float(((low - want).abs() / tolerance(A, S, 40, D, 3)).max()) > 3.0


@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("H,Hkv,D,bs", [(8, 2, 64, 16), (10, 2, 96, 16), (8, 2, 128, 16), (16, 1, 128, 16), (4, 2, 256, 16), (8, 2, 128, 32), (6, 2, 40, 16)])
def test_f32_queries_keep_their_digits(H, Hkv, D, bs, kind, aligned):
    """On the matrix cores and off them: a view off its alignment gives no other digits than half of these allow."""
    from zealot_amd import ops
    lens = [40, 1, 17, 300]
    kp, vp, table, keys, values = problem(D + bs, lens, H, Hkv, D, kind, bs)
    q = between((len(lens), H, D), 7 * D).cuda()
    if not aligned:
        buf = torch.zeros(q.numel() + 1, device="cuda")
        buf[1:] = q.flatten()
        q = buf[1:].view(q.shape)
    ks, vs = [(0.5 + torch.rand(len(lens), Hkv, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (4, 5)]
    scale = 2.0 / D
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), every_page(table, Hkv), scale=scale, k_scales=ks, v_scales=vs)
    assert got.dtype == torch.float32
    check(got, q, keys, values, Hkv, scale, 1 if kind == "f32" else 3, False, ks, vs)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("lens", [[700, 16, 3], [5000]])
def test_weights_keep_their_bits(lens, D, kind):
    """24 for f32 queries (here of few bits, so that neither their rounding nor the output's hides the weights'), 16 for
    bf16 ones; lists in parts too."""
    from zealot_amd import ops
    H, Hkv = 8, 2
    kp, vp, table, keys, values = problem(D, lens, H, Hkv, D, kind, 16)
    q = torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(D)).bfloat16().float().cuda()
    ks, vs = [(0.5 + torch.rand(len(lens), Hkv, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (6, 7)]
    scale = 1 / math.sqrt(D)
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), every_page(table, Hkv), k_scales=ks, v_scales=vs)
    check(got, q, keys, values, Hkv, scale, 3, False, ks, vs)
    low = ops.paged_decode_sparse(q.bfloat16(), kp, vp, table, _ints(lens), every_page(table, Hkv), k_scales=ks, v_scales=vs)
    check(low, q, keys, values, Hkv, scale, 1, True, ks, vs, half=2.0 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_every_page_and_the_dense_decode_agree_by_element(kind):
    """Each within its own tolerance of the same 64-bit rows; the decode over all pages has weights of 8 bits."""
    from zealot_amd import ops
    lens, H, Hkv, D = [700, 100, 64, 1], 32, 8, 128
    kp, vp, table, keys, values = problem(3, lens, H, Hkv, D, kind, 16)
    q = torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    ks, vs = [(0.5 + torch.rand(len(lens), Hkv, generator=torch.Generator().manual_seed(s))).cuda() if kind == "fp8" else None for s in (8, 9)]
    scale = 1 / math.sqrt(D)
    a = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), every_page(table, Hkv), k_scales=ks, v_scales=vs).double().cpu()
    b = ops.paged_decode(q, kp, vp, table, _ints(lens), k_scales=ks, v_scales=vs).double().cpu()
    check(a, q, keys, values, Hkv, scale, 1, True, ks, vs, half=2.0 ** -8)
    for i in range(len(lens)):
        for j in range(H):
            k, v = keys[i][j // 4], values[i][j // 4]
            if ks is not None:
                k, v = k * float(ks[i, j // 4]), v * float(vs[i, j // 4])
            want, A, S = attend64(q[i, j].double().cpu(), k, v, scale)
            tol = tolerance(A, S, len(k), D)
            # the two roundings to bf16 and the other call's weights of 8 bits
            assert bool(((a[i, j] - b[i, j]).abs() <= (2 * tol + 2.0 ** -8 * A) * (1 + 2.0 ** -8) + 2 * 2.0 ** -8 * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_f32_queries_against_infinite_keys_and_values(D):
    """Keys of -inf have weight 0 and infinite values stay infinite, with queries of few digits (parts of zero) and of many."""
    from zealot_amd import ops
    lens, Hkv = [40, 40], 2
    kp, vp, table, keys, values = problem(D, lens, 4, Hkv, D, "bf16", 16)
    q = between((2, 4, D), D).cuda()
    q[0] = 1.0
    want = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), every_page(table, Hkv), scale=2.0 / D)
    for i in range(2):
        b = int(table[i, 1])
        kp[b, :, 3] = float("-inf")
        for h in range(Hkv):
            keep = [t for t in range(40) if t != 19]
            keys[i][h], values[i][h] = keys[i][h][keep], values[i][h][keep]
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), every_page(table, Hkv), scale=2.0 / D)
    assert bool(torch.isfinite(got).all()) and not torch.equal(got, want)
    check(got, q, keys, values, Hkv, 2.0 / D, 3, False)
    q[1, 2, 5] = float("nan")
    q[1, 3, 5] = float("inf")
    vp[int(table[0, 0]), :, 0, 2] = float("inf")
    got = ops.paged_decode_sparse(q, kp, vp, table, _ints(lens), every_page(table, Hkv), scale=2.0 / D)
    assert bool((got[0, :, 2] == float("inf")).all()) and bool(torch.isfinite(got[0, :, 3:]).all())
    assert bool(torch.isnan(got[1, 2:]).all()) and bool(torch.isfinite(got[1, :2]).all())
