"""Rows in 8 bits, 8-bit products and low-rank adapters as they are used together
on the MI355X: the projections of a layer, eager and captured, each checked in 64
bits on what it was really given; and model steps (scheduler, KV cache, chunked
prompts and decode steps in one batch) with 8-bit projections, with requests that
bring adapters, and with both, against the oracle's per-sequence restatement on
each request's own weights W + c B A.

Bars.  f32 with adapters: 2e-4 of the largest |logit|, as without (f32 sums in
another order).  8 bits: a value's rounding to e4m3 is off by 2^-4 / sqrt(3) of its power
of two in the mean square, 2.6 % of the value over a binade; an output of a product
is then off by 2.6 % of its norm.  A layer's qkv gives 2.6 %, gate and up 2.6 % each in
a product of the two (1.2 for SiLU's slope), down 2.6 %: sqrt(1 + 2.9 + 1) x 2.6 % = 5.7 % of the
hidden rows if each counted whole, 8.1 % after two layers.  10^4 logits are off by at
most 4.5 of those standard deviations, and the largest of 512 is 3 of the logits' own: 12 %,
and bf16's 6 % / 2 beside it in the mean square: below 15 %."""
import numpy as np
import pytest
import torch

from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _randn(seed, shape, dtype=F32, by=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * by).to(dtype).cuda()


def _values(rows):
    return rows.data.double() * rows.scales.double()[:, None]


def _product(x, w):
    """(x . w^T in f64, what a bf16 result may be off by)."""
    y = x @ w.t()
    # bf16's half step, and the 8-bit products' 7 x 2^-13 of the sum of magnitudes
    return y, y.abs() * 2.0 ** -8 + 7 * 2.0 ** -13 * (x.abs() @ w.abs().t())


def _rounds_to(q, s, y, off):
    """q, s: rows in 8 bits of y, which is known up to `off`."""
    top, slack = y.abs().amax(1), off.amax(1)
    assert ((s.double() - top / 448).abs() <= slack / 448 + top / 448 * 2.0 ** -17).all()
    # a step of e4m3 is 2^-3 of its power of two, at most 2^-3 of the value, at least 2^-9
    got = q.double() * s.double()[:, None]
    half = torch.maximum(y.abs() * 2.0 ** -4, s.double()[:, None] * 2.0 ** -10)
    assert ((got - y).abs() <= half * (1 + 2.0 ** -3) + 2 * off + y.abs() * 2.0 ** -16).all()


@pytest.mark.parametrize("T,hidden,inter,rank,adapters", [(1, 256, 512, 16, 1), (37, 256, 688, 16, 5), (300, 512, 1024, 8, 3),
                                                         (1100, 256, 512, 32, 4)])
def test_a_layers_projections(T, hidden, inter, rank, adapters):
    from zealot_amd import dense
    x, resid = _randn(1, (T, hidden), BF), _randn(2, (T, hidden), BF)
    nw = (1 + 0.1 * _randn(3, (hidden,))).to(BF)
    W1 = dense.fp8_weight(_randn(4, (2 * inter, hidden), BF, hidden ** -0.5))
    W2 = dense.fp8_weight(_randn(5, (hidden, inter), BF, inter ** -0.5))
    A1, B1 = _randn(6, (adapters, 2 * rank, hidden), BF, hidden ** -0.5), _randn(7, (adapters, 2 * inter, rank), BF, rank ** -0.5)
    A2, B2 = _randn(8, (adapters, rank, inter), BF, inter ** -0.5), _randn(9, (adapters, hidden, rank), BF, rank ** -0.5)
    c = 0.5 + torch.rand(adapters, generator=torch.Generator().manual_seed(10)).cuda()
    ids = torch.randint(-1, adapters, (T,), generator=torch.Generator().manual_seed(11), dtype=torch.int32).cuda()

    def run():
        plan = dense.lora_plan(ids, adapters)
        n, kept = dense.rms_norm_fp8(x, nw, residual=resid)
        base1 = dense.linear_fp8(n, W1)
        gu = dense.lora(n, A1, B1, c, plan, base1.clone(), parts=(inter, inter))
        act = dense.silu_mul_fp8(gu[:, :inter], gu[:, inter:])
        base2 = dense.linear_fp8(act, W2)
        y = dense.lora(act, A2, B2, c, plan, base2.clone())
        return [*n, kept, base1, gu, *act, base2, y]

    got = run()
    nq, ns, kept, base1, gu, aq, as_, base2, y = got
    d = (x.float() + resid.float()).to(BF).double()
    assert torch.equal(kept.double(), d)
    _rounds_to(nq, ns, d * (d.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * nw.double(), torch.zeros_like(d))
    n64, a64 = nq.double() * ns.double()[:, None], aq.double() * as_.double()[:, None]
    for rows, W, out in ((n64, W1, base1), (a64, W2, base2)):
        want, off = _product(rows, W.rowmajor().double() * W.scales.double()[:, None])
        assert ((out.double() - want).abs() <= off).all()

    def added(rows, a, b, base, parts):
        want, off = base.double().clone(), torch.zeros_like(base, dtype=torch.float64)
        width, r = b.shape[1] // parts, b.shape[2]
        for t in range(adapters):
            m = ids == t
            for p in range(parts):
                cols = slice(p * width, (p + 1) * width)
                ap, bp = a[t, p * r:(p + 1) * r].double(), b[t, cols].double()
                v = c[t].double() * (rows[m] @ ap.t())
                want[m, cols] += v @ bp.t()
                # sums in f32 of values held to 2^-16 (two bf16 parts): below 2^-13 of the magnitudes
                off[m, cols] = 2.0 ** -13 * ((c[t].double() * (rows[m].abs() @ ap.abs().t())) @ bp.abs().t())
        return want, off + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8)

    for rows, a, b, base, out, parts in ((n64, A1, B1, base1, gu, 2), (a64, A2, B2, base2, y, 1)):
        want, off = added(rows, a, b, base, parts)
        has = ids >= 0
        assert torch.equal(out[~has], base[~has])
        assert ((out.double() - want).abs() <= off)[has].all()
    g, u = gu[:, :inter].double(), gu[:, inter:].double()
    s = g / (1 + (-g).exp()) * u
    _rounds_to(aq, as_, s, s.abs() * 2.0 ** -18)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        x.copy_(_randn(20 + i, (T, hidden), BF))
        ids.copy_(torch.randint(-1, adapters, (T,), generator=torch.Generator().manual_seed(30 + i), dtype=torch.int32))
        graph.replay()
        eager = run()  # (the graph's buffers are its own)
        torch.cuda.synchronize()
        for u, v in zip(held, eager):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


def _numpy_weights(w, ad, index, cfg):
    """The oracle's weights of a request with adapter `index` (None: none)."""
    from oracle.llama_ref import weights_to_numpy
    from zealot_amd import dense
    from zealot_amd.model import LayerWeights, LlamaWeights
    H, Hkv, D, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.intermediate_size

    def full(t):
        if isinstance(t, dense.Fp8Weight):
            return t.rowmajor().double() * t.scales.double()[:, None]
        return (t if isinstance(t, torch.Tensor) else t.rowmajor()).double()

    def delta(pair, cols):
        if index is None:
            return 0.0
        a, b = pair[0][index].double(), pair[1][index].double()
        r, o, parts = b.shape[1], 0, []
        for p, n in enumerate(cols):
            parts.append(b[o:o + n] @ a[p * r:(p + 1) * r])
            o += n
        return ad.scales[index].double() * torch.cat(parts)

    layers = []
    for i, lw in enumerate(w.layers):
        la = ad.layers[i] if ad is not None else None
        pair = lambda name: getattr(la, name) if la else None  # noqa: E731
        gu = full(lw.gate_up)
        eight = isinstance(lw.gate_up, dense.Fp8Weight)
        gate, up = (gu[:I], gu[I:]) if eight else dense.split_gate_up(gu)
        pg = pair("gate_up")
        if pg and not eight:
            pg = (pg[0], torch.stack([torch.cat(dense.split_gate_up(t)) for t in pg[1]]))
        dg = delta(pg, (I, I))
        merged = dense.interleave_gate_up(*((gate, up) if index is None else (gate + dg[:I], up + dg[I:])))
        f = lambda t: t.float()  # noqa: E731
        layers.append(LayerWeights(lw.attn_norm, f(full(lw.qkv) + delta(pair("qkv"), (H * D, Hkv * D, Hkv * D))),
                                   f(full(lw.o) + delta(pair("o"), (cfg.hidden_size,))), lw.ffn_norm, f(merged),
                                   f(full(lw.down) + delta(pair("down"), (cfg.hidden_size,)))))
    return weights_to_numpy(LlamaWeights(w.embedding, layers, w.final_norm, w.lm_head))


def _serve(dtype, in_8_bits, bring, tol, rope=False):
    """bring: the adapter of each request (None: the runner has none).  Returns the steps' logits."""
    import zealot_amd as ze
    from oracle.llama_ref import LlamaRef
    from zealot_amd import KVCache, PagedKVRunner, Priority, Scheduler, SchedulerConfig
    from zealot_amd.model import HipModelRunner, LlamaAdapters, LlamaConfig, LlamaWeights
    cfg = LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_layers=2, num_heads=8, num_kv_heads=2, head_dim=64,
                      rope_theta=10000.0 if rope else 0.0, max_positions=128 if rope else 0)
    bm = ze.BlockManager(64, 16)
    sched = Scheduler(SchedulerConfig(max_num_seqs=4, block_size=16, num_gpu_blocks=64, max_prefill_tokens=64, prefill_chunk_size=32),
                      block_manager=bm)
    cache = KVCache(64, 16, cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, dtype=dtype, max_seqs=8, max_blocks_per_seq=64)
    w = LlamaWeights.random(cfg, dtype=dtype, seed=11)
    if in_8_bits:
        w = w.in_8_bits()
    ad = LlamaAdapters.random(cfg, 3, 16, dtype, seed=12, in_8_bits=in_8_bits) if bring is not None else None
    runner = HipModelRunner(cfg, w, PagedKVRunner(cache, bm), ad)
    bring = bring or {}
    rng = np.random.default_rng(13)
    prompts, max_new = {"a": 45, "b": 7, "c": 70}, {"a": 6, "b": 9, "c": 4}
    refs = {r: LlamaRef(cfg, _numpy_weights(w, ad, bring.get(r), cfg)) for r in prompts} if tol else {}
    for rid, p in prompts.items():
        sched.add(sched.make_sequence(rid, list(rng.integers(0, cfg.vocab_size, p)), max_new[rid], Priority.Medium))
    worst, all_logits = 0.0, []
    while not sched.is_idle():
        assert len(all_logits) < 100
        out = sched.schedule()
        announce(f"step {len(all_logits)}: {[(e.request_id, e.num_tokens, e.tokens_before) for e in out.batch]}")
        logits = runner.step(out, bring) if bring else runner.step(out)
        all_logits.append(logits.clone())
        logits = logits.cpu().numpy()
        if refs:
            want = np.concatenate([refs[e.request_id].step([(e.request_id, e.step_input(), e.tokens_before)]) for e in out.batch])
            worst = max(worst, float(np.abs(logits - want).max() / np.abs(want).max()))
        for i, e in enumerate(out.batch):
            if not e.is_prefill() or e.is_final_chunk():
                e.push_token(int(rng.integers(0, cfg.vocab_size)))
                if e.is_prefill():
                    e.mark_prefilled()
        for e in out.batch:
            if e.is_prefill():
                sched.advance_prefill(e.request_id)
        for e in out.batch:
            info = sched.seq_info(e.request_id)
            if info["state"] == 1 and info["output_len"] >= max_new[e.request_id]:
                runner.drop_state(e.request_id)
                sched.finish(e.request_id)
    announce(f"worst {worst:.2e} of the largest |logit|")
    assert worst <= (tol or 0), worst
    return all_logits


SOME = {"a": 2, "c": 0}


def test_model_with_adapters_f32():
    _serve(F32, False, SOME, 2e-4)


def test_model_with_adapters_bf16():
    _serve(BF, False, SOME, 6e-2)


def test_model_in_8_bits():
    _serve(BF, True, None, 0.15)


def test_model_in_8_bits_with_adapters():
    _serve(BF, True, SOME, 0.15)


def test_model_whose_requests_bring_no_adapter():
    """Steps without an adapter are what they are without adapters at all."""
    for eight in (False, True):
        plain, none = _serve(BF, eight, None, None), _serve(BF, eight, {}, None)
        assert len(plain) == len(none) and all(torch.equal(u, v) for u, v in zip(plain, none))


def test_model_with_rotated_heads():
    """Both forms go through the rotary KV write too, and adapters change the logits."""
    assert all(t.isfinite().all() for t in _serve(BF, True, SOME, None, rope=True))
    plain, with_b = _serve(F32, False, None, None, rope=True), _serve(F32, False, SOME, None, rope=True)
    assert not torch.equal(plain[0], with_b[0])


def test_adapters_that_are_not_there():
    import zealot_amd as ze
    from zealot_amd import KVCache, PagedKVRunner, Priority, Scheduler, SchedulerConfig
    from zealot_amd.model import HipModelRunner, LlamaAdapters, LlamaConfig, LlamaWeights
    cfg = LlamaConfig(64, 64, 64, 1, 1, 1, 64)
    bm = ze.BlockManager(8, 16)
    sched = Scheduler(SchedulerConfig(max_num_seqs=4, block_size=16, num_gpu_blocks=8), block_manager=bm)
    cache = KVCache(8, 16, 1, 1, 64, dtype=F32, max_seqs=4, max_blocks_per_seq=8)
    w = LlamaWeights.random(cfg, dtype=F32)
    kv = PagedKVRunner(cache, bm)
    with pytest.raises(TypeError):
        w.in_8_bits()
    ad = LlamaAdapters.random(cfg, 2, 4, F32)
    with pytest.raises(ValueError):
        HipModelRunner(cfg, w, kv, LlamaAdapters(2, []))
    with pytest.raises(ValueError):  # gate and up rows in the other order
        HipModelRunner(cfg, w, kv, LlamaAdapters.random(cfg, 2, 4, F32, in_8_bits=True))
    sched.add(sched.make_sequence("a", [1, 2, 3], 2, Priority.Medium))
    out = sched.schedule()
    with pytest.raises(ValueError):
        HipModelRunner(cfg, w, kv).step(out, {"a": 0})
    runner = HipModelRunner(cfg, w, kv, ad)
    for bad in (2, -1):
        with pytest.raises(ValueError):
            runner.step(out, {"a": bad})
    assert runner.step(out, {"a": 1, "other": 9}).shape == (1, 64)
    kv.drop_state("a")
    none = runner.step(out, {"a": None}).clone()
    kv.drop_state("a")
    assert torch.equal(none, HipModelRunner(cfg, w, kv).step(out))
