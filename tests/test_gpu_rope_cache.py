"""KVCache.write_batch_rope and the model with rotary embedding and head norms
on the MI355X.  The cache call is the two calls on the same inputs
(dense.qk_norm_rope, then write_batch), bit for bit on pools of the source's
type; on fp8 pools K is rounded once, so it is held to the formula (half a step,
2^-4, of the value and 24 x 2^-24 of |y_a| + |y_b|, as tests/test_gpu_rope.py
derives).  The model's logits are held to a float64 restatement of its step with
the bars of tests/test_gpu_model.py: 2e-4 of the largest |logit| in f32, 6e-2 in
bf16."""
import numpy as np
import pytest
import torch

from tests.test_gpu_rope import U, _reference

pytestmark = pytest.mark.gpu


def _cache(dtype, layers=2, hkv=2, d=64, blocks=64, scales=None):
    import zealot_amd as ze
    from zealot_amd import KVCache
    bm = ze.BlockManager(blocks, 16)
    c = KVCache(blocks, 16, layers, hkv, d, dtype=dtype, max_seqs=8, max_blocks_per_seq=blocks)
    for rid in ("a", "b", "c"):
        c.register_seq(rid, 32)
        for _ in range(8):
            c.alloc_block(rid, bm)
        if dtype == torch.float8_e4m3fn:
            c.set_fp8_scales(rid, [0.02] * (layers * hkv), [0.03] * (layers * hkv))
    return c, bm


def _step(seed, rows, H, hkv, d, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, (H + 2 * hkv) * d, generator=g).to(dtype).cuda()
    return [t.unflatten(1, (-1, d)) for t in x.split((H * d, hkv * d, hkv * d), 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_cache_call_is_the_two_calls(dtype, interleaved):
    from zealot_amd import dense
    H, hkv, d = 8, 2, 64
    one, _bm1 = _cache(dtype)
    two, _bm2 = _cache(dtype)
    rope = dense.rope_table(128, d)
    g = torch.Generator().manual_seed(1)
    wq, wk = [(1 + 0.1 * torch.randn(d, generator=g)).to(dtype).cuda() for _ in range(2)]
    before = [0, 0, 0]
    for step, counts in enumerate([[20, 0, 3], [1, 5, 1], [1, 1, 1]]):
        T = sum(counts)
        pos = torch.tensor([b + j for b, n in zip(before, counts) for j in range(n)], dtype=torch.int32, device="cuda")
        for layer in range(2):
            q, k, v = _step(10 * step + layer, T, H, hkv, d, dtype)
            want_q, want_k = dense.qk_norm_rope(q, k, pos, rope, wq, wk, interleaved=interleaved)
            two.write_batch(layer, ["a", "b", "c"], counts, want_k, v.contiguous())
            got = one.write_batch_rope(layer, ["a", "b", "c"], counts, q, k, v, rope, wq, wk, interleaved=interleaved, q_out=q)
            torch.cuda.synchronize()
            assert torch.equal(got, want_q) and got.data_ptr() == q.data_ptr()
            assert torch.equal(one.k_pool(layer), two.k_pool(layer)) and torch.equal(one.v_pool(layer), two.v_pool(layer))
            a = one.attention_batch(layer, ["a", "b", "c"], counts, got)
            b = two.attention_batch(layer, ["a", "b", "c"], counts, want_q)
            assert torch.equal(a, b)
        before = [b + n for b, n in zip(before, counts)]
        assert [one.seq_state(r).cached_tokens for r in "abc"] == before


def test_fp8_pools_round_keys_once():
    from zealot_amd import dense
    H, hkv, d = 8, 2, 64
    c, _bm = _cache(torch.float8_e4m3fn)
    rope = dense.rope_table(128, d)
    q, k, v = _step(3, 30, H, hkv, d, torch.bfloat16)
    c.write_batch_rope(0, ["a", "b"], [20, 10], q, k, v, rope)
    pos = torch.tensor(list(range(20)) + list(range(10)), dtype=torch.int32)
    ref, mag = _reference(k, None, pos, rope, False)
    table = [c.seq_state(r).block_ids for r in "ab"]
    pool = c.k_pool(0).float().double().cpu()
    got = torch.stack([pool[table[i][p // 16], :, p % 16] for i, n in enumerate((20, 10)) for p in range(n)])
    ref, mag = ref / float(np.float32(0.02)), mag / 0.02
    assert bool(((got - ref.clamp(-448, 448)).abs() <= 24 * U * mag * 1.0625 + torch.maximum(ref.abs() / 16, torch.tensor(2.0 ** -10))).all())


def test_a_fork_copies_before_its_first_write():
    from zealot_amd import dense
    c, _bm = _cache(torch.bfloat16, layers=1)
    rope = dense.rope_table(128, 64)
    q, k, v = _step(4, 20, 8, 2, 64, torch.bfloat16)
    c.write_batch_rope(0, ["a"], [20], q, k, v, rope)
    c.release_seq("b")
    c.fork_seq("a", "b")
    q, k, v = _step(5, 2, 8, 2, 64, torch.bfloat16)
    c.write_batch_rope(0, ["a", "b"], [1, 1], q, k, v, rope)
    ta, tb = c.seq_state("a").block_ids, c.seq_state("b").block_ids
    assert ta[0] == tb[0] and ta[1] != tb[1]
    want = dense.qk_norm_rope(q, k, torch.full((2,), 20, dtype=torch.int32, device="cuda"), rope)[1]
    pool = c.k_pool(0)
    assert torch.equal(pool[ta[1], :, 4], want[0]) and torch.equal(pool[tb[1], :, 4], want[1])
    assert torch.equal(pool[ta[1], :, :4], pool[tb[1], :, :4])


def test_refusals_change_nothing():
    from zealot_amd import ZealotError, _lib, dense
    c, _bm = _cache(torch.bfloat16, layers=1)
    rope = dense.rope_table(30, 64)
    q, k, v = _step(6, 20, 8, 2, 64, torch.bfloat16)
    c.write_batch_rope(0, ["a"], [20], q, k, v, rope)
    c.release_seq("b")
    c.fork_seq("a", "b")
    torch.cuda.synchronize()
    pool, tables = c.k_pool(0).clone(), (c.seq_state("a").block_ids, c.seq_state("b").block_ids)
    q, k, v = _step(7, 11, 8, 2, 64, torch.bfloat16)
    with pytest.raises(ZealotError) as e:  # position 30 of 30
        c.write_batch_rope(0, ["b"], [11], q, k, v, rope)
    assert e.value.code == _lib.ERR_SEQUENCE_TOO_LONG and e.value.fields == {"required": 31, "capacity": 30}
    with pytest.raises(ZealotError):  # K's rows as the query output
        c.write_batch_rope(0, ["b"], [2], q[:2], k[:2], v[:2], rope, q_out=torch.as_strided(k, (2, 8, 64), k.stride()))
    with pytest.raises(ValueError):
        c.write_batch_rope(0, ["b"], [2], q[:2], k[:2], v[:2], rope, q_weight=torch.ones(63, dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(c.k_pool(0), pool) and tables == (c.seq_state("a").block_ids, c.seq_state("b").block_ids)
    c.write_batch_rope(0, ["b"], [10], q[:10], k[:10], v[:10], rope)
    assert c.seq_state("b").cached_tokens == 30


class _Ref:
    """The model's step in float64, sequence by sequence."""

    def __init__(self, cfg, w):
        full = lambda t: (t.rowmajor() if hasattr(t, "rowmajor") else t).double().cpu()  # noqa: E731
        from zealot_amd.dense import split_gate_up
        self.cfg, self.kv = cfg, {}
        self.emb, self.final, self.head = full(w.embedding), full(w.final_norm), full(w.lm_head)
        self.layers = []
        for lw in w.layers:
            gate, up = split_gate_up(lw.gate_up.rowmajor() if hasattr(lw.gate_up, "rowmajor") else lw.gate_up)
            self.layers.append(dict(an=full(lw.attn_norm), qkv=full(lw.qkv), o=full(lw.o), fn=full(lw.ffn_norm), gate=full(gate), up=full(up),
                                    down=full(lw.down), qn=None if lw.q_norm is None else full(lw.q_norm),
                                    kn=None if lw.k_norm is None else full(lw.k_norm)))

    def _norm(self, x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.cfg.rms_eps) * w

    def _turn(self, x, pos):
        c = self.cfg
        D = c.head_dim
        if c.rope_theta <= 0:
            return x
        angle = pos[:, None, None] * c.rope_theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        a, b = (x[..., 0::2], x[..., 1::2]) if c.rope_interleaved else (x[..., :D // 2], x[..., D // 2:])
        a, b = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
        return torch.stack([a, b], -1).flatten(-2) if c.rope_interleaved else torch.cat([a, b], -1)

    def step(self, entries):
        c = self.cfg
        H, hkv, D = c.num_heads, c.num_kv_heads, c.head_dim
        out = []
        for rid, ids, before in entries:
            h = self.emb[torch.tensor(ids)]
            pos = torch.arange(before, before + len(ids), dtype=torch.float64)
            for i, lw in enumerate(self.layers):
                x = self._norm(h, lw["an"]) @ lw["qkv"].t()
                q, k, v = [t.unflatten(1, (-1, D)) for t in x.split((H * D, hkv * D, hkv * D), 1)]
                if c.qk_norm:
                    q, k = self._norm(q, lw["qn"]), self._norm(k, lw["kn"])
                q, k = self._turn(q, pos), self._turn(k, pos)
                if before:
                    k, v = torch.cat([self.kv[rid, i][0], k]), torch.cat([self.kv[rid, i][1], v])
                self.kv[rid, i] = k, v
                kk, vv = k.repeat_interleave(H // hkv, 1), v.repeat_interleave(H // hkv, 1)
                s = torch.einsum("thd,shd->hts", q, kk) / D ** 0.5
                s = s.masked_fill(torch.arange(k.shape[0]) > pos[:, None], float("-inf"))
                att = torch.einsum("hts,shd->thd", torch.softmax(s, 2), vv).flatten(1)
                h = h + att @ lw["o"].t()
                x = self._norm(h, lw["fn"])
                g = x @ lw["gate"].t()
                h = h + (g * torch.sigmoid(g) * (x @ lw["up"].t())) @ lw["down"].t()
            out.append(self._norm(h[-1], self.final) @ self.head.t())
        return torch.stack(out)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 6e-2)])
@pytest.mark.parametrize("theta,inter,norm", [(10000.0, False, True), (500000.0, True, False), (0.0, False, True)])
def test_model_step(dtype, tol, theta, inter, norm):
    import zealot_amd as ze
    from zealot_amd import KVCache, PagedKVRunner, Scheduler, SchedulerConfig
    from zealot_amd.model import HipModelRunner, LlamaConfig, LlamaWeights
    cfg = LlamaConfig(512, 256, 512, 2, 8, 2, 64, rope_theta=theta, max_positions=256, rope_interleaved=inter, qk_norm=norm)
    bm = ze.BlockManager(64, 16)
    sched = Scheduler(SchedulerConfig(max_num_seqs=4, block_size=16, num_gpu_blocks=64, max_prefill_tokens=64, prefill_chunk_size=32),
                      block_manager=bm)
    cache = KVCache(64, 16, cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, dtype=dtype, max_seqs=8, max_blocks_per_seq=64)
    w = LlamaWeights.random(cfg, dtype=dtype, seed=11)
    runner, ref = HipModelRunner(cfg, w, PagedKVRunner(cache, bm)), _Ref(cfg, w)
    rng = np.random.default_rng(12)
    for rid, n in {"a": 45, "b": 7, "c": 70}.items():
        sched.add(sched.make_sequence(rid, list(rng.integers(0, cfg.vocab_size, n)), 4, ze.Priority.Medium))
    steps = 0
    while not sched.is_idle():
        steps += 1
        assert steps < 50
        out = sched.schedule()
        entries = [(e.request_id, e.step_input(), e.tokens_before) for e in out.batch]
        logits = runner.step(out).double().cpu()
        want = ref.step(entries)
        assert float((logits - want).abs().max()) <= tol * float(want.abs().max())
        for i, e in enumerate(out.batch):
            if not e.is_prefill() or e.is_final_chunk():
                e.push_token(int(logits[i].argmax()))
                if e.is_prefill():
                    e.mark_prefilled()
        for e in out.batch:
            if e.is_prefill():
                sched.advance_prefill(e.request_id)
        for e in out.batch:
            info = sched.seq_info(e.request_id)
            if info["state"] == 1 and info["output_len"] >= 4:
                runner.drop_state(e.request_id)
                sched.finish(e.request_id)


def test_a_default_model_draws_the_same_weights():
    """The new fields change nothing of a model without them."""
    from zealot_amd.model import LlamaConfig, LlamaWeights
    cfg = LlamaConfig(64, 128, 128, 1, 2, 1, 64)
    a = LlamaWeights.random(cfg, dtype=torch.float32, seed=3)
    b = LlamaWeights.random(LlamaConfig(64, 128, 128, 1, 2, 1, 64, rope_theta=10000.0, max_positions=8), dtype=torch.float32, seed=3)
    assert torch.equal(a.lm_head, b.lm_head) and torch.equal(a.layers[0].down, b.layers[0].down) and a.layers[0].q_norm is None
