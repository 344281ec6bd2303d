"""A row's norm and rotation is the same, bit for bit, whatever the call's other
operands are: their alignment and strides, how many heads share the call, and
whether K goes to a tensor or to a pool of the source's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = [torch.float32, torch.bfloat16]
# (heads, kv-heads, head size, rotated dimensions)
SHAPES = [(32, 8, 128, 128), (6, 2, 64, 64), (20, 4, 96, 96), (4, 2, 128, 64), (3, 1, 256, 256), (70, 2, 64, 64), (2, 1, 17, 16), (3, 2, 34, 30)]


def _problem(seed, T, H, Hkv, D, rot, dtype):
    from zealot_amd import dense
    g = torch.Generator().manual_seed(seed)
    x = {"q": torch.randn(T, H, D, generator=g), "k": torch.randn(T, Hkv, D, generator=g), "v": torch.randn(T, Hkv, D, generator=g)}
    x = {n: t.to(dtype).cuda() for n, t in x.items()}
    x["q_weight"], x["k_weight"] = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2)]
    x["rope"] = dense.rope_table(300, rot)
    x["positions"] = torch.randint(0, 300, (T,), generator=g, dtype=torch.int32).cuda()
    x["slots"] = torch.randperm((T // 16 + 2) * 16, generator=g)[:T].cuda()
    x["k_pool"], x["v_pool"] = [torch.zeros(T // 16 + 2, Hkv, 16, D, dtype=dtype, device="cuda") for _ in range(2)]
    return x


def _off(t):
    """The same values one element behind a vector's border."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    buf[1:] = t.flatten()
    return buf[1:].view(t.shape)


def _odd_rows(t):
    """The same rows, an odd number of elements apart."""
    buf = torch.empty(t.shape[0], t.shape[1] * t.shape[2] + 1, dtype=t.dtype, device="cuda")
    buf[:, :-1] = t.flatten(1)
    return buf[:, :-1].unflatten(1, t.shape[1:])


def _fused(x, interleaved):
    from zealot_amd import ops
    kp, vp = x["k_pool"], x["v_pool"]
    kp.zero_()
    vp.zero_()
    q = ops.qk_norm_rope_append(kp, vp, x["q"], x["k"], x["v"], x["positions"], x["slots"], x["rope"], x["q_weight"], x["k_weight"],
                                interleaved=interleaved, q_out=x.get("q_out"))
    return q.clone(), kp.clone(), vp.clone()


def _separate(x, interleaved):
    from zealot_amd import dense, ops
    kp, vp = torch.zeros_like(x["k_pool"]), torch.zeros_like(x["v_pool"])
    q, k = dense.qk_norm_rope(x["q"], x["k"], x["positions"], x["rope"], x["q_weight"], x["k_weight"], interleaved=interleaved,
                              q_out=x.get("q_out"), k_out=x.get("k_out"))
    ops.append(kp, vp, k.contiguous(), x["v"].contiguous(), x["slots"])
    return q.clone(), kp, vp


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hkv,D,rot", SHAPES)
def test_alignment_and_strides(H, Hkv, D, rot, interleaved, dtype):
    x = _problem(H + D, 37, H, Hkv, D, rot, dtype)
    want = _fused(x, interleaved)
    for got in (_separate(x, interleaved),):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for name in ("q", "k", "v", "q_weight", "k_weight", "rope", "k_pool", "v_pool", "q_out", "k_out", "q/", "k/", "v/", "q_out/"):
        y = dict(x)
        if name.startswith("q_out"):
            y["q_out"] = torch.empty_like(x["q"])
        if name == "k_out":
            y["k_out"] = _off(torch.empty_like(x["k"]))
        elif name.endswith("/"):
            y[name[:-1]] = _odd_rows(y[name[:-1]])
        else:
            y[name] = _off(y[name])
        for call in (_fused, _separate):
            got = call(y, interleaved)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (name, call.__name__)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_other_heads_of_the_call(interleaved, dtype):
    """One head's rows alone, and among enough heads and tokens for every number of heads a lane."""
    from zealot_amd import dense
    T = 2500
    for H, Hkv in ((8, 2), (24, 8), (40, 8), (56, 8), (72, 8)):
        x = _problem(H, T, H, Hkv, 128, 128, dtype)
        how = dict(interleaved=interleaved)
        q, k = dense.qk_norm_rope(x["q"], x["k"], x["positions"], x["rope"], x["q_weight"], x["k_weight"], **how)
        one = dense.qk_norm_rope(x["q"][:, :1], x["k"][:, :1], x["positions"], x["rope"], x["q_weight"], x["k_weight"], **how)
        assert torch.equal(q[:, :1], one[0]) and torch.equal(k[:, :1], one[1])
        got = _fused(x, interleaved)
        assert torch.equal(got[0], q) and torch.equal(got[1].transpose(1, 2).flatten(0, 1)[x["slots"]], k)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("which", [(True, False), (False, True), (False, False)])
def test_without_weights_or_a_table(which, dtype):
    x = _problem(5, 30, 6, 2, 128, 128, dtype)
    for name, on in zip(("q_weight", "k_weight"), which):
        if not on:
            x[name] = None
    for table in (x["rope"], None):
        x["rope"] = table
        want = _fused(x, False)
        for name in ("q", "v", "v_pool"):
            y = dict(x)
            y[name] = _off(y[name])
            for call in (_fused, _separate):
                assert all(torch.equal(a, b) for a, b in zip(call(y, False), want)), (name, call.__name__)


@pytest.mark.parametrize("pool", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("dtype", KINDS)
def test_pools_of_other_types(dtype, pool):
    """Off their alignment and on it: the same bytes."""
    from zealot_amd import ops
    T, H, Hkv, D = 50, 4, 2, 64
    x = _problem(6, T, H, Hkv, D, D, dtype)
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}[pool]
    more = {}
    if pool == "fp8":
        more = dict(k_scales=torch.full((2, Hkv), 0.02, device="cuda"), v_scales=torch.full((2, Hkv), 0.03, device="cuda"),
                    token_row=(torch.arange(T, dtype=torch.int32) % 2).cuda())
    outs = []
    for off in (False, True):
        n = x["k_pool"].numel()
        raw = [torch.zeros(n + 1, device="cuda").to(t) for _ in range(2)]
        kp, vp = [r[int(off):n + int(off)].view(x["k_pool"].shape) for r in raw]
        q = ops.qk_norm_rope_append(kp, vp, x["q"], x["k"], x["v"], x["positions"], x["slots"], x["rope"], x["q_weight"], x["k_weight"], **more)
        outs.append((q, kp.contiguous().view(torch.uint8) if pool == "fp8" else kp, vp.contiguous().view(torch.uint8) if pool == "fp8" else vp))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", KINDS)
def test_norms_alone_through_the_cache(dtype, kind):
    """Without a table the cache's call takes no positions: the two calls' bits, step after step, with a plain write between."""
    import zealot_amd as ze
    from zealot_amd import KVCache, dense
    H, hkv, d, ids = 4, 2, 64, ["a", "b"]
    caches, managers = [], []  # (a cache's blocks belong to its manager)
    for _ in range(2):
        bm, c = ze.BlockManager(32, 16), KVCache(32, 16, 1, hkv, d, dtype=kind, max_seqs=4, max_blocks_per_seq=16)
        for rid in ids:
            c.register_seq(rid, 16)
            for _ in range(8):
                c.alloc_block(rid, bm)
            if kind == torch.float8_e4m3fn:
                c.set_fp8_scales(rid, [0.02] * hkv, [0.03] * hkv)
        caches.append(c)
        managers.append(bm)
    g = torch.Generator().manual_seed(3)
    wq, wk = [(1 + 0.1 * torch.randn(d, generator=g)).to(dtype).cuda() for _ in range(2)]
    for step, counts in enumerate([[20, 3], [1, 40], [1, 1], [5, 0], [1, 1]]):
        T = sum(counts)
        q, k, v = [torch.randn(T, h, d, generator=g).to(dtype).cuda() for h in (H, hkv, hkv)]
        if step == 3:  # as projected
            for c in caches:
                c.write_batch(0, ids, counts, k, v)
            continue
        got = caches[0].write_batch_rope(0, ids, counts, q, k, v, None, wq, wk)
        # K's one rounding is to the pool's type: equal where the separate calls' K is f32, or of the pool's type
        if kind == dtype or dtype == torch.float32:
            want_q, want_k = dense.qk_norm_rope(q, k, None, None, wq, wk)
            caches[1].write_batch(0, ids, counts, want_k, v)
            assert torch.equal(got, want_q)
            torch.cuda.synchronize()
            for a, b in ((caches[0].k_pool(0), caches[1].k_pool(0)), (caches[0].v_pool(0), caches[1].v_pool(0))):
                for i, rid in enumerate(ids):
                    rows = [c.seq_state(rid) for c in caches]
                    assert rows[0].cached_tokens == rows[1].cached_tokens
                    x, y = [p.view(torch.uint8)[torch.tensor(r.block_ids, device="cuda")].transpose(1, 2).flatten(0, 1)[:r.cached_tokens]
                            for p, r in zip((a, b), rows)]
                    assert torch.equal(x, y), (step, rid)
        else:
            torch.cuda.synchronize()


def test_a_sequence_without_new_tokens_may_lie_behind_the_table():
    """Written as projected past the table's positions, then in a batch of rotated keys with no token of its own."""
    import zealot_amd as ze
    from zealot_amd import KVCache, ZealotError, dense
    H, hkv, d = 4, 2, 64
    bm, c = ze.BlockManager(16, 16), KVCache(16, 16, 1, hkv, d, dtype=torch.bfloat16, max_seqs=4, max_blocks_per_seq=8)
    for rid in "ab":
        c.register_seq(rid, 4)
        for _ in range(4):
            c.alloc_block(rid, bm)
    rope = dense.rope_table(30, d)
    q, k, v = [torch.randn(40, h, d, dtype=torch.bfloat16, device="cuda") for h in (H, hkv, hkv)]
    c.write_batch(0, ["a"], [40], k, v)
    got = c.write_batch_rope(0, ["a", "b"], [0, 5], q[:5], k[:5], v[:5], rope)
    want = dense.qk_norm_rope(q[:5], k[:5], torch.arange(5, dtype=torch.int32, device="cuda"), rope)[0]
    assert torch.equal(got, want) and c.seq_state("a").cached_tokens == 40 and c.seq_state("b").cached_tokens == 5
    with pytest.raises(ZealotError) as e:
        c.write_batch_rope(0, ["a", "b"], [1, 5], q[:6], k[:6], v[:6], rope)
    assert e.value.fields == {"required": 41, "capacity": 30}
    assert "seq a would hold 41 tokens" in str(e.value) and "30 rows" in str(e.value) and "blocks" not in str(e.value)
