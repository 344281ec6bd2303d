"""A batched Llama-shaped ModelRunner step on the gfx950 path: the dense ops
(zealot_amd.dense) around one KV write and one attention call per layer for
the whole schedule() batch.

Same math as the reference runner's step (src/cuda_runner.rs:271-660):
embedding -> per layer [RMSNorm -> q/k/v projections -> KV store -> paged
attention -> o_proj -> residual add -> RMSNorm -> gate/up projections ->
SiLU(gate) * up -> down projection -> residual add] -> final RMSNorm of each
sequence's last token -> lm_head logits.  The reference has no rotary
embedding and no norms of the heads, and neither has a model by default; with
rope_theta or qk_norm set, both run in the KV write's launch
(PagedKVRunner.write_rope).  What differs is the shape of the work:
  - one launch per op for all sequences of the batch (the reference loops
    over sequences, cuda_runner.rs:274);
  - q/k/v come from ONE projection against a fused [(H + 2 Hkv) D, hidden]
    weight (its split-k sums, when it has them, added by the kernel that
    writes K and V to the pages: zk_cache_write_batch_qkv), gate/up from one
    against [2 I, hidden] whose gate and up rows
    alternate in blocks of 16, so the projection's waves hold the gate and
    up outputs of the same columns and write SiLU(gate) * up themselves
    (dense.linear_silu_mul); K and V are appended and
    q attended straight out of the fused output through row strides (no
    transpose kernels, no copies; cf. cuda_runner.rs:373-392);
  - each residual add is fused into the RMSNorm that follows it, and so,
    for the o and down projections, is the projection's split-k sum when it
    runs on the weight-streaming kernel (dense.linear_rms_norm); the final
    norm runs only over the last row of each sequence;
  - the large decode-time weights (gate|up, down, lm_head) are kept tiled
    (dense.TiledWeight): the weight-streaming kernel reads them with
    contiguous 1 KiB loads; their row-major copies serve steps of more than
    64 rows (prefill, mixed) on the GEMM plan, since the weight-streaming
    kernel reads a weight once per 64 rows;
  - with projections in 8 bits (LlamaWeights.in_8_bits: qkv, gate|up and down) the
    norms and SiLU * up write the rows that the 8-bit products read (rms_norm_fp8,
    silu_mul_fp8, linear_fp8); the o projection, whose rows attention writes, and
    lm_head stay in bf16;
  - requests may bring low-rank adapters (LlamaAdapters, step's `adapters`): the
    rows of a step are grouped by adapter once (lora_plan) and each projection
    adds its rows' adapters to its output (lora).  A step without any runs as
    before;
  - weights are random-initialised here (there is no checkpoint loader in
    this build; the reference loads HF weights, model_loader.rs:241).
"""
from __future__ import annotations

import math
import operator
from dataclasses import dataclass, replace

import torch

from . import dense
from .runner import PagedKVRunner, StepPlan


@dataclass
class LlamaConfig:
    vocab_size: int
    hidden_size: int
    intermediate_size: int
    num_layers: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    rms_eps: float = 1e-6
    rope_theta: float = 0.0       # base of the rotary embedding's frequencies; 0: none
    max_positions: int = 0        # rows of its table
    rope_interleaved: bool = False  # pairs (2 i, 2 i + 1) instead of (i, i + head_dim / 2)
    qk_norm: bool = False         # RMSNorm of every query and key head

    @staticmethod
    def llama3_8b(num_layers: int = 32) -> "LlamaConfig":
        return LlamaConfig(128256, 4096, 14336, num_layers, 32, 8, 128)


@dataclass
class LayerWeights:
    attn_norm: torch.Tensor  # [hidden]
    qkv: torch.Tensor        # [(H + 2 Hkv) D, hidden]: q rows, then k, then v
    o: torch.Tensor          # [hidden, H D]
    ffn_norm: torch.Tensor   # [hidden]
    gate_up: object          # [2 I, hidden]: gate and up rows interleaved in blocks of 16 (dense.interleave_gate_up);
                             # a dense.TiledWeight of it for bf16 models
    down: object             # [hidden, I] (a dense.TiledWeight for bf16 models)
    q_norm: torch.Tensor | None = None  # [head_dim], of models with qk_norm
    k_norm: torch.Tensor | None = None


def _check_8_bits(lw: LayerWeights) -> None:
    """The rows that the layer's 8-bit projections read can be written."""
    for what, k in (("hidden", lw.qkv.shape[1]), ("hidden", lw.gate_up.shape[1]), ("intermediate", lw.down.shape[1])):
        if k % 16 or k > dense.FP8_LONGEST_ROW:
            raise ValueError(f"8-bit projections need a {what} size that is a multiple of 16 up to {dense.FP8_LONGEST_ROW}, not {k}")


@dataclass
class LlamaWeights:
    embedding: torch.Tensor  # [vocab, hidden]
    layers: list
    final_norm: torch.Tensor  # [hidden]
    lm_head: object           # [vocab, hidden] (a dense.TiledWeight for bf16 models)

    def in_8_bits(self) -> "LlamaWeights":
        """The model with qkv, gate|up and down as dense.Fp8Weight (bf16 models
        whose hidden and intermediate sizes are multiples of 16 up to
        dense.FP8_LONGEST_ROW): gate|up holds the gate rows, then the up rows.
        The rest is shared."""
        if self.embedding.dtype != torch.bfloat16:
            raise TypeError("8-bit projections are for bf16 models")
        if any(isinstance(lw.gate_up, dense.Fp8Weight) for lw in self.layers):
            raise ValueError("the projections are in 8 bits already")
        for lw in self.layers:
            _check_8_bits(lw)

        def full(t):
            return t if isinstance(t, torch.Tensor) else t.rowmajor() if t.full is None else t.full

        def layer(lw):
            gate_up = torch.cat(dense.split_gate_up(full(lw.gate_up)))
            return replace(lw, qkv=dense.fp8_weight(full(lw.qkv)), gate_up=dense.fp8_weight(gate_up),
                           down=dense.fp8_weight(full(lw.down)))
        return replace(self, layers=[layer(lw) for lw in self.layers])

    @staticmethod
    def random(cfg: LlamaConfig, dtype=torch.bfloat16, device="cuda", seed: int = 0,
               tiled: bool = True, keep_full: bool = True) -> "LlamaWeights":
        """N(0, 1/fan_in) projections and N(1, 0.1) norm weights (seeded);
        with tiled (bf16 only) gate|up, down and lm_head as dense.TiledWeight,
        keeping their row-major copies for steps of more than 64 rows unless
        keep_full is off (decode-only callers: half the memory of those
        weights)."""
        g = torch.Generator(device=device).manual_seed(seed)
        tile = ((lambda t: dense.tile_weight(t, keep_full=keep_full)) if tiled and dtype == torch.bfloat16
                else (lambda t: t))

        def lin(n, k):
            return (torch.randn((n, k), generator=g, device=device) / math.sqrt(k)).to(dtype)

        def norm(n):
            return (1 + 0.1 * torch.randn((n,), generator=g, device=device)).to(dtype)

        H, Hkv, D, hid, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.hidden_size, cfg.intermediate_size
        layers = [LayerWeights(norm(hid), lin((H + 2 * Hkv) * D, hid), lin(hid, H * D), norm(hid),
                               tile(dense.interleave_gate_up(lin(I, hid), lin(I, hid))), tile(lin(hid, I)))
                  for _ in range(cfg.num_layers)]
        if cfg.qk_norm:
            for lw in layers:
                lw.q_norm, lw.k_norm = norm(D), norm(D)
        emb = torch.randn((cfg.vocab_size, hid), generator=g, device=device).to(dtype)
        return LlamaWeights(emb, layers, norm(hid), tile(lin(cfg.vocab_size, hid)))


@dataclass
class LayerAdapters:
    """One layer's adapters for dense.lora: (a, b) of each projection, or None."""
    qkv: tuple | None = None      # a [A, 3 r, hidden] (q, k and v ranks), b [A, (H + 2 Hkv) D, r]
    o: tuple | None = None        # a [A, r, H D], b [A, hidden, r]
    gate_up: tuple | None = None  # a [A, 2 r, hidden], b [A, 2 I, r] in the rows' order of the model's gate_up
    down: tuple | None = None     # a [A, r, I], b [A, hidden, r]


@dataclass
class LlamaAdapters:
    """The low-rank adapters that requests may name, of the model's type."""
    count: int
    layers: list
    scales: torch.Tensor | None = None  # float32 [count]; None: 1
    in_8_bits: bool = False  # for a model of LlamaWeights.in_8_bits, whose gate and up rows do not alternate

    def check(self, cfg: LlamaConfig, like: torch.Tensor) -> None:
        """Raises unless dense.lora takes these adapters beside the projections of a
        model of this shape and of `like`'s type and device."""
        H, Hkv, D, hid, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.hidden_size, cfg.intermediate_size
        shapes = {"qkv": (3, (H + 2 * Hkv) * D, hid), "o": (1, hid, H * D), "gate_up": (2, 2 * I, hid), "down": (1, hid, I)}

        def need(t, name, shape, dtype):
            if not isinstance(t, torch.Tensor) or t.dtype != dtype:
                raise TypeError(f"{name} of the adapters must be {dtype}")
            if tuple(t.shape) != shape or not t.is_contiguous() or t.device != like.device:
                raise ValueError(f"{name} of the adapters must be a contiguous {list(shape)} on {like.device}")

        if self.scales is not None:
            need(self.scales, "scales", (self.count,), torch.float32)
        for i, layer in enumerate(self.layers):
            for name, (parts, n, k) in shapes.items():
                pair = getattr(layer, name)
                if pair is None:
                    continue
                a, b = pair
                rank = b.shape[-1]
                need(a, f"layer {i}: a of {name}", (self.count, parts * rank, k), like.dtype)
                need(b, f"layer {i}: b of {name}", (self.count, n, rank), like.dtype)
                if dense.lora_workspace_bytes(1, self.count, k, rank, parts, like.dtype) == 0:
                    raise ValueError(f"layer {i}: {self.count} adapters of rank {rank} for {name} ({parts} parts) are more than dense.lora takes")

    @staticmethod
    def random(cfg: LlamaConfig, count: int, rank: int, dtype=torch.bfloat16, device="cuda", seed: int = 0,
               in_8_bits: bool = False) -> "LlamaAdapters":
        """N(0, 1/fan_in) a and b, for every projection (seeded)."""
        g = torch.Generator(device=device).manual_seed(seed)

        def mat(n, k):
            return (torch.randn((count, n, k), generator=g, device=device) / math.sqrt(k)).to(dtype)

        def pair(n, k, parts=1):
            return mat(parts * rank, k), mat(n, rank)

        def gate_up(n, k):
            a, b = pair(2 * n, k, 2)
            if not in_8_bits:
                b = torch.stack([dense.interleave_gate_up(t[:n], t[n:]) for t in b])
            return a, b

        H, Hkv, D, hid, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.hidden_size, cfg.intermediate_size
        layers = [LayerAdapters(pair((H + 2 * Hkv) * D, hid, 3), pair(hid, H * D), gate_up(I, hid), pair(hid, I))
                  for _ in range(cfg.num_layers)]
        return LlamaAdapters(count, layers, 0.5 + torch.rand((count,), generator=g, device=device), in_8_bits)


class HipModelRunner:
    """ModelRunner::step (engine.rs:15-37) for a schedule() batch: returns the
    f32 logits [len(batch), vocab] of each sequence's last step token."""

    def __init__(self, cfg: LlamaConfig, weights: LlamaWeights, kv: PagedKVRunner, adapters: LlamaAdapters | None = None):
        c = kv.cache
        if (c.num_layers, c.num_kv_heads, c.head_dim) != (cfg.num_layers, cfg.num_kv_heads, cfg.head_dim):
            raise ValueError("KV cache shape does not match the model")
        self.cfg, self.w, self.kv = cfg, weights, kv
        self.rope = None
        if cfg.rope_theta > 0:
            self.rope = dense.rope_table(cfg.max_positions, cfg.head_dim, cfg.rope_theta, weights.embedding.device)
        if cfg.qk_norm and any(lw.q_norm is None or lw.k_norm is None for lw in weights.layers):
            raise ValueError("a model with qk_norm needs the layers' q_norm and k_norm")
        # what a step would refuse is refused here: a step that fails half way has written to the cache
        eight = [isinstance(t, dense.Fp8Weight) for lw in weights.layers for t in (lw.qkv, lw.gate_up, lw.down)]
        self.in_8_bits = any(eight)
        if self.in_8_bits:
            if not all(eight):
                raise ValueError("qkv, gate_up and down of every layer must be in 8 bits, or none")
            for lw in weights.layers:
                _check_8_bits(lw)
        if adapters is not None and (len(adapters.layers) != len(weights.layers) or adapters.in_8_bits != self.in_8_bits):
            raise ValueError("adapters must have the model's layers, and gate and up rows in its order (in_8_bits)")
        if adapters is not None:
            adapters.check(cfg, weights.embedding)
        self.adapters = adapters

    def drop_state(self, request_id: str) -> None:
        self.kv.drop_state(request_id)

    def step(self, out, adapters: dict | None = None) -> torch.Tensor:
        """One step over ScheduleOutput `out` (zealot_amd.scheduler); adapters:
        the adapter of each request id that brings one (others: none, or None), the
        same at all its steps."""
        per_row = self._adapter_rows(out, adapters)
        plan = self.kv.begin_step(out)
        if not out.batch:
            return torch.empty((0, self.cfg.vocab_size), dtype=torch.float32, device=self.w.embedding.device)
        # ids and last rows in one upload from pinned memory: the host does not
        # wait for it, so the layers' calls run ahead of the device
        ids = [t for e in out.batch for t in e.step_input()]
        both = torch.tensor(ids + plan_last_rows(plan), dtype=torch.int64, pin_memory=True)
        both = both.to(self.w.embedding.device, non_blocking=True)
        lora = None
        if per_row is not None:
            rows = torch.tensor(per_row, dtype=torch.int32, pin_memory=True)
            lora = dense.lora_plan(rows.to(both.device, non_blocking=True), self.adapters.count)
        return self.forward(plan, both[:len(ids)], both[len(ids):], lora)

    def _adapter_rows(self, out, adapters: dict | None):
        """The adapter of every step row (-1: none), or None where no row has one."""
        ids = [e.request_id for e in out.batch] if adapters else []
        # (operator.index: a whole number, or TypeError)
        mine = {rid: operator.index(adapters[rid]) for rid in ids if adapters.get(rid) is not None}
        if not mine:
            return None
        if self.adapters is None:
            raise ValueError("the runner has no adapters")
        for rid, a in mine.items():
            if not 0 <= a < self.adapters.count:
                raise ValueError(f"request {rid} names adapter {a} of {self.adapters.count}")
        return [mine.get(e.request_id, -1) for e in out.batch for _ in range(e.num_tokens)]

    def _norm(self, x, weight, resid=None):
        """The norm of x, or of resid += x, as the next projection reads it."""
        eps = self.cfg.rms_eps
        norm = dense.rms_norm_fp8 if self.in_8_bits else dense.rms_norm
        return norm(x, weight, eps) if resid is None else norm(x, weight, eps, residual=resid, residual_out=resid)[0]

    def _forward_apart(self, plan: StepPlan, ids: torch.Tensor, last_rows: torch.Tensor, lora) -> torch.Tensor:
        """forward with each projection on its own: in 8 bits, or with the rows'
        adapters added before its output is used."""
        cfg, w, T = self.cfg, self.w, plan.total_tokens
        H, Hkv, D, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.intermediate_size
        qd, kd = H * D, Hkv * D

        def project(x, weight, adapters, **parts):
            y = dense.linear_fp8(x, weight) if isinstance(weight, dense.Fp8Weight) else dense.linear(x, weight)
            if adapters is not None:
                dense.lora(x, *adapters, self.adapters.scales, lora, y, **parts)
            return y

        resid = dense.embedding(ids, w.embedding)
        normed = self._norm(resid, w.layers[0].attn_norm)
        for layer, lw in enumerate(w.layers):
            ad = LayerAdapters() if lora is None else self.adapters.layers[layer]
            qkv = project(normed, lw.qkv, ad.qkv, parts=(qd, kd, kd))
            q, k, v = (t.view(T, -1, D) for t in qkv.split((qd, kd, kd), 1))
            if self.rope is not None or cfg.qk_norm:
                self.kv.write_rope(layer, plan, q, k, v, self.rope, lw.q_norm if cfg.qk_norm else None,
                                   lw.k_norm if cfg.qk_norm else None, cfg.rms_eps, cfg.rope_interleaved, q_out=q)
            else:
                self.kv.write(layer, plan, k, v)
            attn = self.kv.attention(layer, plan, q)
            normed = self._norm(project(attn.view(T, qd), lw.o, ad.o), lw.ffn_norm, resid)
            if self.in_8_bits:
                gu = project(normed, lw.gate_up, ad.gate_up, parts=(I, I))
                act = dense.silu_mul_fp8(gu[:, :I], gu[:, I:])
            else:  # gate and up columns alternate in blocks: a block is a row of SiLU's
                b = dense.GATE_UP_BLOCK
                gu = project(normed, lw.gate_up, ad.gate_up, parts=2, part_block=b).view(-1, 2 * b)
                act = dense.silu_mul(gu[:, :b], gu[:, b:]).view(T, I)
            delta = project(act, lw.down, ad.down)
            if layer + 1 < len(w.layers):
                normed = self._norm(delta, w.layers[layer + 1].attn_norm, resid)
        final, _ = dense.rms_norm(delta, w.final_norm, cfg.rms_eps, residual=resid, rows=last_rows)
        return dense.linear(final, w.lm_head, out_dtype=torch.float32)

    def forward(self, plan: StepPlan, ids: torch.Tensor, last_rows: torch.Tensor, lora=None) -> torch.Tensor:
        """The step's logits; lora: the dense.lora_plan of its rows' adapters."""
        cfg, w = self.cfg, self.w
        if ids.numel() != plan.total_tokens:
            raise ValueError("one token id per step row")
        if lora is not None and self.adapters is None:
            raise ValueError("the runner has no adapters")
        if lora is not None or self.in_8_bits:
            return self._forward_apart(plan, ids, last_rows, lora)
        H, Hkv, D = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
        T = plan.total_tokens
        qd, kd = H * D, Hkv * D
        resid = dense.embedding(ids, w.embedding)  # the residual stream [T, hidden]
        normed = torch.empty_like(resid)
        dense.rms_norm(resid, w.layers[0].attn_norm, cfg.rms_eps, out=normed)
        last = len(w.layers) - 1
        for layer, lw in enumerate(w.layers):
            if self.rope is not None or cfg.qk_norm:  # heads normalised and rotated on the way to the pages
                qkv = dense.linear(normed, lw.qkv)
                q = qkv[:, :qd].view(T, H, D)
                self.kv.write_rope(layer, plan, q, qkv[:, qd:qd + kd].view(T, Hkv, D), qkv[:, qd + kd:].view(T, Hkv, D),
                                   self.rope, lw.q_norm if cfg.qk_norm else None, lw.k_norm if cfg.qk_norm else None,
                                   cfg.rms_eps, cfg.rope_interleaved, q_out=q)
            elif normed.dtype == torch.bfloat16:  # projection and KV write in one call
                qkv = self.kv.write_qkv(layer, plan, normed, lw.qkv, H)
            else:
                qkv = dense.linear(normed, lw.qkv)
                self.kv.write(layer, plan, qkv[:, qd:qd + kd].view(T, Hkv, D), qkv[:, qd + kd:].view(T, Hkv, D))
            q = qkv[:, :qd].view(T, H, D)
            attn = self.kv.attention(layer, plan, q)
            # resid += o_proj(attn); normed = norm(resid)
            dense.linear_rms_norm(attn.view(T, qd), lw.o, lw.ffn_norm, cfg.rms_eps, residual=resid, out=normed,
                                  residual_out=resid)
            act = dense.linear_silu_mul(normed, lw.gate_up)
            if layer < last:  # resid += down_proj(act); normed = the next layer's attention norm of resid
                dense.linear_rms_norm(act, lw.down, w.layers[layer + 1].attn_norm, cfg.rms_eps, residual=resid,
                                      out=normed, residual_out=resid)
        delta = dense.linear(act, w.layers[last].down)
        final, _ = dense.rms_norm(delta, w.final_norm, cfg.rms_eps, residual=resid, rows=last_rows)
        return dense.linear(final, w.lm_head, out_dtype=torch.float32)


def plan_last_rows(plan: StepPlan) -> list:
    """Row of each entry's last step token in the packed batch."""
    rows, o = [], 0
    for n in plan.num_tokens[:len(plan.ids)]:
        o += int(n)
        rows.append(o - 1)
    return rows
