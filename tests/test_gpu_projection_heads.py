"""Model steps with rotary embedding and head norms whose projections stand alone
(requests with adapters, 8-bit weights) on the MI355X: adapters before the norm and the
rotation, on the parts that they belong to.

f32 and bf16: logits against the same scheduler run of a plain f32 model on each
request's own weights W + c B A, within the bars of test_gpu_projection_run.py (2e-4 of
the largest |logit|, 6e-2).

8 bits: stage by stage in 64 bits on what each was given, since the logits of a model with
adapters as large as its weights move by 0.1 to 0.35 of the largest from the rows'
rounding to e4m3 alone.  q, k and v of the first layer: the product's bounds (a bf16
result's half step, 7 x 2^-13 of the sum of magnitudes), the adapters' (2^-13 of theirs) and
the half step of the second rounding.  Normed and rotated heads: bf16's half step
and f32's steps of the terms (16 x 2^-24, and 2^-22 for the table's angles).  Attention: weights,
output and keys rounded to bf16, each 2^-8 of the largest value at most: 2^-6."""
import numpy as np
import pytest
import torch

from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _full(t):
    from zealot_amd import dense
    if isinstance(t, dense.Fp8Weight):
        return t.rowmajor().double() * t.scales.double()[:, None]
    return (t if isinstance(t, torch.Tensor) else t.rowmajor()).double()


def _own_weights(w, ad, i, cfg):
    """A plain f32 model's weights: w, and with i the adapter added to them."""
    from zealot_amd import dense
    from zealot_amd.model import LayerWeights, LlamaWeights
    H, Hkv, D, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.intermediate_size

    def merged(t, pair, part):
        t = _full(t)
        if i is None:
            return t
        a, b = pair[0][i].double(), pair[1][i].double()
        r = b.shape[1]
        for p in range(a.shape[0] // r):
            mine = part == p
            t[mine] += ad.scales[i].double() * b[mine] @ a[p * r:(p + 1) * r]
        return t

    one = torch.zeros(cfg.hidden_size, dtype=torch.int64, device="cuda")
    qkv = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor([H * D, Hkv * D, Hkv * D], device="cuda"))
    layers = []
    for n, lw in enumerate(w.layers):
        la = ad.layers[n]
        eight = isinstance(lw.gate_up, dense.Fp8Weight)
        rows = torch.arange(2 * I, device="cuda")
        gu = merged(lw.gate_up, la.gate_up, rows // I if eight else rows // dense.GATE_UP_BLOCK % 2)
        if eight:
            gu = dense.interleave_gate_up(gu[:I], gu[I:])
        f = lambda t: None if t is None else t.float().contiguous()  # noqa: E731
        layers.append(LayerWeights(f(lw.attn_norm), f(merged(lw.qkv, la.qkv, qkv)), f(merged(lw.o, la.o, one)), f(lw.ffn_norm), f(gu),
                                   f(merged(lw.down, la.down, one)), f(lw.q_norm), f(lw.k_norm)))
    return LlamaWeights(w.embedding.float(), layers, w.final_norm.float(), _full(w.lm_head).float())


def _serve(cfg, w, dtype, ad=None, bring=None, kind=None, each=None):
    """[{request: logits}] of a run with chunked prompts and decode steps; its tokens are drawn, not taken from the logits.
    kind: of the KV runner; each(runner, batch) is called behind every step."""
    import zealot_amd as ze
    from zealot_amd import KVCache, PagedKVRunner, Priority, Scheduler, SchedulerConfig
    from zealot_amd.model import HipModelRunner
    bm = ze.BlockManager(64, 16)
    sched = Scheduler(SchedulerConfig(max_num_seqs=4, block_size=16, num_gpu_blocks=64, max_prefill_tokens=64, prefill_chunk_size=32),
                      block_manager=bm)
    cache = KVCache(64, 16, cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, dtype=dtype, max_seqs=8, max_blocks_per_seq=64)
    runner = HipModelRunner(cfg, w, (kind or PagedKVRunner)(cache, bm), ad)
    rng = np.random.default_rng(3)
    max_new = {"a": 5, "b": 8, "c": 4}
    for rid, p in {"a": 45, "b": 7, "c": 70}.items():
        sched.add(sched.make_sequence(rid, list(rng.integers(0, cfg.vocab_size, p)), max_new[rid], Priority.Medium))
    steps = []
    while not sched.is_idle():
        assert len(steps) < 100
        out = sched.schedule()
        announce(f"step {len(steps)}: {[(e.request_id, e.num_tokens, e.tokens_before) for e in out.batch]}")
        logits = runner.step(out, bring).double()
        steps.append({e.request_id: logits[i] for i, e in enumerate(out.batch)})
        if each:
            each(runner, out.batch)
        for e in out.batch:
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
    return steps


BRING = {"a": 2, "c": 0}  # (b: none)


HEADS = [(True, False, False), (True, True, True), (False, False, True)]


def _config(rope, interleaved, qk_norm):
    from zealot_amd.model import LlamaConfig
    return LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_layers=2, num_heads=8, num_kv_heads=2, head_dim=64,
                       rope_theta=10000.0 if rope else 0.0, max_positions=128 if rope else 0, rope_interleaved=interleaved, qk_norm=qk_norm)


@pytest.mark.parametrize("dtype,bar", [(F32, 2e-4), (BF, 6e-2)])
@pytest.mark.parametrize("rope,interleaved,qk_norm", HEADS)
def test_adapters_under_head_norms_and_rotation(rope, interleaved, qk_norm, dtype, bar):
    from zealot_amd.model import LlamaAdapters, LlamaWeights
    cfg = _config(rope, interleaved, qk_norm)
    w = LlamaWeights.random(cfg, dtype=dtype, seed=21)
    ad = LlamaAdapters.random(cfg, 3, 16, dtype, seed=22)
    got = _serve(cfg, w, dtype, ad, BRING)
    want = {rid: _serve(cfg, _own_weights(w, ad, BRING.get(rid), cfg), F32) for rid in "abc"}
    worst = 0.0
    for i, step in enumerate(got):
        for rid, logits in step.items():
            ref = want[rid][i][rid]
            worst = max(worst, float((logits - ref).abs().max() / ref.abs().max()))
    announce(f"worst {worst:.2e} of the largest |logit|")
    assert worst <= bar, worst


def _heads(x, pos, weight, cfg):
    """(heads [T, n, D] as the pages and attention have them, in f64; what they may be off by)."""
    D, rope = cfg.head_dim, cfg.rope_theta > 0
    y = x.double()
    if weight is not None:
        y = y * (y.pow(2).mean(-1, keepdim=True) + cfg.rms_eps).rsqrt() * weight.double()
    off = 16 * 2.0 ** -24 * y.abs()
    if rope:
        i = torch.arange(D // 2, device="cuda", dtype=torch.float64)
        angle = pos.double()[:, None, None] * cfg.rope_theta ** (-2 * i / D)
        first, second = (slice(0, None, 2), slice(1, None, 2)) if cfg.rope_interleaved else (slice(0, D // 2), slice(D // 2, None))
        u, v, out = y[..., first], y[..., second], torch.empty_like(y)
        out[..., first], out[..., second] = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
        most = torch.empty_like(y)
        most[..., first] = most[..., second] = u.abs() + v.abs()
        y, off = out, (16 * 2.0 ** -24 + 2.0 ** -22) * most
    return y, off + 2.0 ** -8 * y.abs()


@pytest.mark.parametrize("rope,interleaved,qk_norm", HEADS)
def test_8_bit_heads_stage_by_stage(rope, interleaved, qk_norm):
    from zealot_amd import PagedKVRunner, dense
    from zealot_amd.model import LlamaAdapters, LlamaWeights
    cfg = _config(rope, interleaved, qk_norm)
    w = LlamaWeights.random(cfg, dtype=BF, seed=21).in_8_bits()
    ad = LlamaAdapters.random(cfg, 3, 16, BF, seed=22, in_8_bits=True)
    H, Hkv, D, layers = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, w.layers
    cols = (H * D, Hkv * D, Hkv * D)
    seen = []  # of one step, a layer: [q, k, v as projected, q as attended, attention]
    pages = {}  # (request, layer): keys and values so far

    class Recorder(PagedKVRunner):
        def write_rope(self, layer, plan, q, k, v, *args, **kw):
            seen.append([t.clone() for t in (q, k, v)])
            return super().write_rope(layer, plan, q, k, v, *args, **kw)

        def attention(self, layer, plan, q):
            out = super().attention(layer, plan, q)
            seen[-1] += [q.clone(), out.clone()]
            return out

    def check(runner, batch):
        assert len(seen) == cfg.num_layers
        ids = torch.tensor([t for e in batch for t in e.step_input()], device="cuda")
        pos = torch.cat([e.tokens_before + torch.arange(e.num_tokens, device="cuda") for e in batch])
        n = dense.rms_norm_fp8(dense.embedding(ids, w.embedding), layers[0].attn_norm, cfg.rms_eps)
        n = n.data.double() * n.scales.double()[:, None]
        W, (a, b) = _full(layers[0].qkv), ad.layers[0].qkv
        base, mags = n @ W.T, n.abs() @ W.abs().T
        got, row = torch.cat([t.flatten(1) for t in seen[0][:3]], 1).double(), 0
        for e in batch:
            rows = slice(row, row + e.num_tokens)
            row += e.num_tokens
            want, off = base[rows].clone(), 7 * 2.0 ** -13 * mags[rows] + 2.0 ** -8 * base[rows].abs()
            i, at = BRING.get(e.request_id), 0
            for p, width in enumerate(cols if i is not None else ()):
                ap, bp, c = a[i, 16 * p:16 * (p + 1)].double(), b[i, at:at + width].double(), float(ad.scales[i])
                want[:, at:at + width] += c * (n[rows] @ ap.T) @ bp.T
                off[:, at:at + width] += 2.0 ** -13 * c * (n[rows].abs() @ ap.abs().T) @ bp.abs().T
                at += width
            assert ((got[rows] - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()
        for layer, (q, k, v, q_out, out) in enumerate(seen):
            lw = layers[layer]
            y, off = _heads(q, pos, lw.q_norm, cfg)
            assert ((q_out.double() - y).abs() <= off).all()
            keys, row = _heads(k, pos, lw.k_norm, cfg)[0].bfloat16(), 0
            for e in batch:
                rows = slice(row, row + e.num_tokens)
                row += e.num_tokens
                kv = pages.setdefault((e.request_id, layer), [keys[:0], v[:0]])
                kv[0], kv[1] = torch.cat([kv[0], keys[rows]]), torch.cat([kv[1], v[rows]])
                K, V = (t.double().repeat_interleave(H // Hkv, 1).permute(1, 2, 0) for t in kv)
                s = torch.stack([q_out[rows, h].double() @ K[h] for h in range(H)], 1) / D ** 0.5
                s = s.masked_fill((torch.arange(K.shape[2], device="cuda") > pos[rows, None])[:, None], float("-inf"))
                p = s.softmax(-1)
                want = torch.stack([p[:, h] @ V[h].T.contiguous() for h in range(H)], 1)
                assert ((out.reshape(-1, H, D)[rows].double() - want).abs() <= 2.0 ** -6 * V.abs().max()).all()
        seen.clear()

    _serve(cfg, w, BF, ad, BRING, Recorder, check)
    assert len(pages) == 3 * cfg.num_layers
