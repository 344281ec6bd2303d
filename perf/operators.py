"""Performance cases of the operators around a paged cache whose queries and keys are normalised and rotated and whose
long contexts are attended sparsely: what one layer of a serving step calls, from the step's request lengths to the
attention of its new tokens.

A case is a dict of plain values; `kind` names the operator:

  tables   ops.step_tables: block tables, slot map, positions and offsets of a step from its request lengths
  rope     dense.qk_norm_rope, ops.qk_norm_rope_append: norms of the query and key heads and the position rotation in one
           pass over a fused projection's output, with the write of K and V into the pages (`pool`) or without
  bounds   ops.page_bounds: smallest and largest key of each page and dimension, kept up to date behind a KV write
  scores   ops.page_scores: an upper bound of every page's attention logits for a query, from those bounds
  select   ops.select_pages: the pages of the best scores, with the first and the newest ones
  sparse   ops.paged_decode_sparse: attention of one query row per sequence over its selected pages

Every size and the draw of the lengths (`lens_seed`) belong to the case, the values to the seed.  32 / 8 heads of 128
with 16-token blocks is the shape of the repository's benchmark, 256 contexts of 512 to 8192 tokens its decode batch
and 64 chunks of 512 its prefill batch.
"""
import math
import random

import torch

own = False

BS = 16  # tokens per block
GQA = {"heads": 32, "kv_heads": 8, "dim": 128}
_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f32": 4, "fp8": 1}
EPS = 1e-6


def listed():
    return [
        # a decode step of the full batch: one token each, a new block where a context has just filled its last one
        dict(name="tables_decode", kind="tables", seqs=256, lo=512, hi=8192, new_lo=1, new_hi=1, pad=0, lens_seed=1),
        # a prefill step: 64 chunks of up to 512 tokens, every block of a chunk newly granted
        dict(name="tables_chunks", kind="tables", seqs=64, lo=0, hi=4095, new_lo=300, new_hi=512, pad=100, lens_seed=2),
        # that decode step's queries and keys of one layer, out of the fused projection and into the pages
        dict(name="rope_decode", kind="rope", rows=256, chunk=1, norm=True, interleaved=False, rot=128, max_pos=8192, src="bf16", pool="bf16",
             lens_seed=3, **GQA),
        # those of the full prefill batch
        dict(name="rope_chunks", kind="rope", rows=32768, chunk=512, norm=True, interleaved=False, rot=128, max_pos=8192, src="bf16", pool="bf16",
             lens_seed=4, **GQA),
        # one token each behind the decode step's write: the pages that it went to
        dict(name="bounds_decode", kind="bounds", seqs=256, new_lo=1, new_hi=1, kv="bf16", lens_seed=5, **GQA),
        # a prefill batch's pages
        dict(name="bounds_chunks", kind="bounds", seqs=64, new_lo=300, new_hi=512, kv="bf16", lens_seed=6, **GQA),
        # the decode batch's pages, scored for its queries
        dict(name="scores_batch", kind="scores", seqs=256, lo=512, hi=8192, kv="bf16", q="bf16", mapping="grouped", lens_seed=7, **GQA),
        # two users with long documents
        dict(name="scores_long", kind="scores", seqs=2, lo=100000, hi=131072, kv="fp8", q="bf16", mapping="grouped", lens_seed=8, **GQA),
        # 1024 tokens out of each context of the decode batch
        dict(name="select_batch", kind="select", seqs=256, lo=512, hi=8192, kv_heads=8, pages=64, sink=1, recent=2, lens_seed=9),
        # 4096 tokens out of the two long ones
        dict(name="select_long", kind="select", seqs=2, lo=100000, hi=131072, kv_heads=8, pages=256, sink=1, recent=2, lens_seed=10),
        # the decode batch's attention over the selected pages
        dict(name="sparse_batch", kind="sparse", seqs=256, lo=512, hi=8192, pages=64, kv="bf16", q="bf16", mapping="grouped", lens_seed=11,
             **GQA),
        # the two long contexts', on fp8 pools
        dict(name="sparse_long", kind="sparse", seqs=2, lo=100000, hi=131072, pages=256, kv="fp8", q="bf16", mapping="grouped",
             lens_seed=12, **GQA),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng):
    return rng.choice([GQA, GQA, {"heads": 32, "kv_heads": 32, "dim": 128}, {"heads": 16, "kv_heads": 8, "dim": 64},
                       {"heads": 64, "kv_heads": 8, "dim": 128}, {"heads": 20, "kv_heads": 4, "dim": 96}])


def _context(rng, tokens):
    """Sequences and the range of their contexts, of at most `tokens` in all."""
    seqs = _log_int(rng, 1, 256)
    hi = _log_int(rng, 20, min(131072, max(21, tokens // seqs)))
    return dict(seqs=seqs, lo=rng.choice([0, hi // 16, hi // 2]), hi=hi)


def draw(rng):
    kind = rng.choice(["tables", "rope", "rope", "bounds", "scores", "select", "sparse", "sparse"])
    base = {"kind": kind, "lens_seed": rng.randrange(1 << 20)}
    if kind == "tables":
        seqs = _log_int(rng, 1, 512)
        hi = _log_int(rng, 1, max(1, min(2000, 20000 // seqs)))
        return dict(base, seqs=seqs, lo=0, hi=_log_int(rng, 1, 8192), new_lo=rng.choice([0, 1, max(1, hi // 4)]), new_hi=hi,
                    pad=rng.choice([0, 0, 37]))
    if kind == "rope":
        s = _shape(rng)
        src = rng.choice(["bf16", "bf16", "f32"])
        rows = _log_int(rng, 1, 8000)
        return dict(base, rows=rows, chunk=rng.choice([1, 100, 512]), norm=rng.choice([True, True, False]), interleaved=rng.choice([False, False, True]),
                    rot=rng.choice([s["dim"], s["dim"], s["dim"] // 2]), max_pos=rng.choice([4096, 131072]), src=src,
                    pool=rng.choice(["none", src, "fp8"]), **s)
    if kind == "bounds":
        seqs = _log_int(rng, 1, 256)
        hi = _log_int(rng, 1, max(1, min(1000, 16000 // seqs)))
        return dict(base, seqs=seqs, new_lo=max(1, hi // 4), new_hi=hi, kv=rng.choice(["bf16", "fp8", "f32"]), **_shape(rng))
    if kind == "select":
        c = _context(rng, 500000)
        most = -(-c["hi"] // BS)
        return dict(base, **c, kv_heads=rng.choice([1, 4, 8]), pages=_log_int(rng, 4, max(5, min(512, most + 8))), sink=rng.choice([0, 1, 2]),
                    recent=rng.choice([1, 2]))
    s = _shape(rng)
    kv = rng.choice(["bf16", "bf16", "fp8", "f32"])
    c = _context(rng, 800000 * 8 // max(8, s["kv_heads"]) * 2 // max(2, _BYTES[kv]))
    base = dict(base, **c, kv=kv, q="f32" if kv == "f32" else "bf16", mapping=rng.choice(["grouped", "grouped", "modulo"]), **s)
    if kind == "scores":
        return base
    room = 16384 * 8 * 128 * 2 // (c["seqs"] * s["kv_heads"] * s["dim"] * max(2, _BYTES[kv]))
    return dict(base, pages=_log_int(rng, 1, max(2, min(512, room, c["hi"] // BS + 2))))


# ------------------------------------------------------------------ sizes and values

def _randint(rng, lo, hi):
    return rng.randint(min(lo, hi), hi)


def _lens(case):
    """(tokens before the step, tokens of the step) of each sequence, or (contexts, None)."""
    rng = random.Random(case["lens_seed"])
    if "new_lo" in case:
        new = [_randint(rng, case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
        return [_randint(rng, case.get("lo", 0), case.get("hi", 4095)) for _ in new], new
    return [_randint(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])], None


def _pages(tokens):
    return -(-tokens // BS)


def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed(seed * 64 + tag)


def _normal(seed, tag, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=_gen(seed, tag), device="cuda", dtype=torch.bfloat16 if dtype != "f32" else torch.float32)
    return (x * scale).to(_TORCH[dtype])


def _permutation(seed, tag, n):
    return torch.randperm(n, generator=_gen(seed, tag), device="cuda").to(torch.int32)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _tables(seed, lens, most=None):
    """Block tables of shuffled blocks, padded with -1, and the pool's number of blocks."""
    pages = _ints([_pages(n) for n in lens], torch.int64)
    total, width = sum(_pages(n) for n in lens), max(1, most or max(_pages(n) for n in lens))
    blocks = _permutation(seed, 1, total + 3)
    at = torch.arange(width, device="cuda")
    first = pages.cumsum(0) - pages
    table = torch.where(at < pages[:, None], blocks[(first[:, None] + at).clamp(max=total)], -1)
    return table.to(torch.int32), total + 3


def _rope_table(max_pos, rot):
    """Cosines, then sines, of every position: angles in 64 bits."""
    freq = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if kind == "tables":
        before, new = _lens(case)
        need = [_pages(b + n) - _pages(b) for b, n in zip(before, new)]
        most = max(1, max(_pages(b + n) for b, n in zip(before, new)))
        s["tables"], blocks = _tables(seed, before, most)
        s["blocks"] = blocks + _permutation(seed, 2, sum(need) + 5)  # granted for this step
        s["seq_lens"], s["new_lens"] = _ints(before), _ints(new)
        s["rows"] = sum(new) + case["pad"]  # a batch is padded to its graph's rows
        return s
    H, Hkv, D = case.get("heads"), case["kv_heads"], case.get("dim")
    if kind == "rope":
        T, src = case["rows"], case["src"]
        s["qkv"] = _normal(seed, 3, (T, (H + 2 * Hkv) * D), src)
        s["rope"] = _rope_table(case["max_pos"], case["rot"])
        # sequences of `chunk` tokens behind others, the last one shorter
        chunk, at = case["chunk"], torch.arange(T, device="cuda")
        seqs, seq, j = -(-T // chunk), at // chunk, at % chunk
        first = torch.randint(0, case["max_pos"] - chunk, (seqs,), generator=_gen(seed, 4), device="cuda")
        s["positions"] = (first[seq] + j).to(torch.int32)
        s["wq"], s["wk"] = [(1 + _normal(seed, t, (D,), "f32", 0.1)).to(_TORCH[src]) if case["norm"] else None for t in (5, 6)]
        if case["pool"] != "none":
            each = _pages(chunk) + 1
            nb = seqs * each + 3
            tib = first[seq] % BS + j
            s["slots"] = _permutation(seed, 7, nb)[seq * each + tib // BS].long() * BS + tib % BS
            s["k_pool"], s["v_pool"] = [torch.zeros((nb, Hkv, BS, D), device="cuda").to(_TORCH[case["pool"]]) for _ in range(2)]
            if case["pool"] == "fp8":  # one scale a sequence and head
                s["k_scales"], s["v_scales"] = [0.01 + 0.01 * torch.rand((seqs, Hkv), generator=_gen(seed, t), device="cuda") for t in (8, 9)]
                s["token_row"] = seq.to(torch.int32)
        return s
    if kind == "bounds":
        before, new = _lens(case)
        table, nb = _tables(seed, [b + n for b, n in zip(before, new)])
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new, torch.int64))
        first = _ints(new, torch.int64).cumsum(0) - _ints(new, torch.int64)
        pos = _ints(before, torch.int64)[seq] + torch.arange(sum(new), device="cuda") - first[seq]
        # the pools of the touched pages alone, renumbered: what the pass reads and writes lies in them
        page = table[seq, pos // BS].long()
        used, page = torch.unique(page, return_inverse=True)
        nb = used.numel() + 3
        s["slots"] = page * BS + pos % BS
        s["k_pool"] = _normal(seed, 3, (nb, Hkv, BS, D), case["kv"])
        b = _normal(seed, 4, (2, nb, Hkv, D), case["kv"]).float()
        s["bounds"] = torch.stack([b.amin(0), b.amax(0)], 2).to(_TORCH[case["kv"]])
        return s
    lens, _ = _lens(case)
    s["seq_lens"] = _ints(lens)
    width = max(1, max(_pages(n) for n in lens))
    if kind == "select":
        x = torch.randn((len(lens), Hkv, width), generator=_gen(seed, 3), device="cuda")
        x = (x * 32).round() / 32 + 5  # equal scores among them
        s["scores"] = torch.where(torch.arange(width, device="cuda") * BS < s["seq_lens"][:, None, None], x, -math.inf)
        return s
    s["tables"], nb = _tables(seed, lens)
    s["q"] = _normal(seed, 3, (len(lens), H, D), case["q"])
    if kind == "scores":
        c, r = _normal(seed, 4, (nb, Hkv, D), "f32", 0.3), _normal(seed, 5, (nb, Hkv, D), "f32", 0.3)
        s["bounds"] = torch.stack([c - 1.6 - r.abs(), c + 1.6 + r.abs()], 2).to(_TORCH[case["kv"]])
        return s
    s["k_pool"], s["v_pool"] = [_normal(seed, t, (nb, Hkv, BS, D), case["kv"]) for t in (4, 5)]
    if case["kv"] == "fp8":
        s["k_scales"], s["v_scales"] = [0.5 + torch.rand((len(lens), Hkv), generator=_gen(seed, t), device="cuda") for t in (6, 7)]
    # pages as a selection gives them: in ascending order, the first and the newest among them, then -1
    held = (s["seq_lens"][:, None, None] + BS - 1) // BS
    at = torch.arange(width, device="cuda")
    x = torch.rand((len(lens), Hkv, width), generator=_gen(seed, 8), device="cuda")
    x = torch.where((at == 0) | (at == held - 1), 2.0, x)
    x = torch.where(at < held, x, -1.0)
    k = min(case["pages"], width)
    best, page = x.topk(k, 2)
    page = torch.where(best >= 0, page, width + 1).sort(2).values
    page = torch.where(page > width, -1, page)
    s["pages"] = torch.cat([page, page.new_full((len(lens), Hkv, case["pages"] - k), -1)], 2).to(torch.int32).contiguous()
    return s


# ------------------------------------------------------------------ one pass

def _split(s):
    c = s["case"]
    T, H, Hkv, D = c["rows"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"]
    return x[:, :H * D].view(T, H, D), x[:, H * D:(H + Hkv) * D].view(T, Hkv, D), x[:, (H + Hkv) * D:].view(T, Hkv, D)


def _run_own(s):
    from zealot_amd import dense, ops

    c, kind = s["case"], s["case"]["kind"]
    if kind == "tables":
        t = ops.step_tables(s["tables"], s["seq_lens"], s["new_lens"], BS, s["rows"], new_blocks=s["blocks"])
        return {"tables": s["tables"], "slots": t.slot_mapping, "positions": t.positions, "rows": t.token_row, "cu": t.cu_seqlens,
                "lens": t.kv_lens, "cursor": t.cursor}
    if kind == "rope":
        q, k, v = _split(s)
        how = dict(q_weight=s["wq"], k_weight=s["wk"], eps=EPS, interleaved=c["interleaved"])
        if c["pool"] == "none":
            q, k = dense.qk_norm_rope(q, k, s["positions"], s["rope"], **how)
            return {"q": q, "k": k}
        q = ops.qk_norm_rope_append(s["k_pool"], s["v_pool"], q, k, v, s["positions"], s["slots"], s["rope"], k_scales=s.get("k_scales"),
                                    v_scales=s.get("v_scales"), token_row=s.get("token_row"), **how)
        return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if kind == "bounds":
        ops.page_bounds(s["k_pool"], s["slots"], s["bounds"])
        return s["bounds"]
    if kind == "scores":
        return ops.page_scores(s["q"], s["bounds"], s["tables"], s["seq_lens"], BS, mapping=c["mapping"])
    if kind == "select":
        return ops.select_pages(s["scores"], s["seq_lens"], BS, c["pages"], sink=c["sink"], recent=c["recent"])
    return ops.paged_decode_sparse(s["q"], s["k_pool"], s["v_pool"], s["tables"], s["seq_lens"], s["pages"], mapping=c["mapping"],
                                   k_scales=s.get("k_scales"), v_scales=s.get("v_scales"))


def _plain_tables(s):
    tables, before, new, blocks = s["tables"], s["seq_lens"].long(), s["new_lens"].long(), s["blocks"]
    width = tables.shape[1]
    after = before + new
    p0, p1 = (before + BS - 1) // BS, (after + BS - 1) // BS
    base = (p1 - p0).cumsum(0) - (p1 - p0)
    at = torch.arange(width, device=tables.device)
    take = (base[:, None] + at - p0[:, None]).clamp(0, blocks.numel() - 1)
    tables = torch.where((at >= p0[:, None]) & (at < p1[:, None]), blocks[take], tables)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["rows"], device=tables.device)
    row = torch.searchsorted(cu[1:], t, right=True)
    real = row < new.numel()
    row = row.clamp(max=new.numel() - 1)
    pos = before[row] + t - cu[row]
    slot = tables[row, (pos // BS).clamp(0, width - 1)].long() * BS + pos % BS
    return {"tables": tables, "slots": torch.where(real, slot, -1), "positions": torch.where(real, pos, -1).int(),
            "rows": torch.where(real, row, -1).int(), "cu": cu, "lens": after.int(), "cursor": (p1 - p0).sum().view(1)}


def _rotated(x, w, cos, sin, interleaved, eps):
    """x [T, heads, D] normalised over D (with a weight) and its first 2 * cos.shape[1] dimensions rotated."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + eps) * w
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], 3).flatten(2) if interleaved else torch.cat([a, b], 2)
    return torch.cat([r, rest], 2)


def _rope_values(s, dtype):
    """(q, k, v) rotated, in `dtype`."""
    c = s["case"]
    q, k, v = [x.to(dtype) for x in _split(s)]
    wq, wk = [None if w is None else w.to(dtype) for w in (s["wq"], s["wk"])]
    half = c["rot"] // 2
    cs = s["rope"][s["positions"].long()].to(dtype)
    cos, sin = cs[:, :half], cs[:, half:]
    return _rotated(q, wq, cos, sin, c["interleaved"], EPS), _rotated(k, wk, cos, sin, c["interleaved"], EPS), v


def _plain_rope(s):
    c = s["case"]
    src = _TORCH[c["src"]]
    q, k, v = _rope_values(s, torch.float32)
    if c["pool"] == "none":
        return {"q": q.to(src), "k": k.to(src)}
    if c["pool"] == "fp8":
        row = s["token_row"].long()
        k, v = [(x * (1 / sc[row])[:, :, None]).clamp(-448, 448) for x, sc in ((k, s["k_scales"]), (v, s["v_scales"]))]
    block, tib = s["slots"] // BS, s["slots"] % BS
    byte = torch.uint8 if c["pool"] == "fp8" else _TORCH[c["pool"]]
    for pool, x in ((s["k_pool"], k), (s["v_pool"], v)):
        pool.view(byte)[block, :, tib] = x.to(_TORCH[c["pool"]]).view(byte)
    return {"q": q.to(src), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_bounds(s):
    pool, slots, old = s["k_pool"], s["slots"], s["bounds"]
    nb, Hkv, _, D = pool.shape
    block = slots // BS
    rows = pool.float()[block, :, slots % BS]
    began = torch.zeros(nb + 1, dtype=torch.bool, device=pool.device)
    began[torch.where(slots % BS == 0, block, nb)] = True  # (row nb: of no block)
    began = began[:nb, None, None]
    at = block[:, None, None].expand_as(rows)
    lo = torch.where(began, math.inf, old[:, :, 0].float()).scatter_reduce(0, at, rows, "amin")
    hi = torch.where(began, -math.inf, old[:, :, 1].float()).scatter_reduce(0, at, rows, "amax")
    return torch.stack([lo, hi], 2).to(old.dtype)


def _heads(case, device):
    """[kv_heads, heads a kv-head]: the query heads of each kv-head."""
    H, Hkv = case["heads"], case["kv_heads"]
    h = torch.arange(H, device=device)
    return h.view(Hkv, H // Hkv) if case["mapping"] == "grouped" else h.view(H // Hkv, Hkv).t()


def _plain_scores(s, dtype=torch.float32):
    tables, lens = s["tables"], s["seq_lens"]
    b = s["bounds"][tables.clamp(min=0).long()].to(dtype)  # [N, pages, Hkv, 2, D]
    q = s["q"].to(dtype)[:, _heads(s["case"], tables.device)]  # [N, Hkv, G, D]
    both = torch.cat([q.clamp(max=0), q.clamp(min=0)], 3)  # what meets the smallest, then the largest key
    x = torch.matmul(b.flatten(3).permute(0, 2, 1, 3).contiguous(), both.transpose(2, 3).contiguous()).amax(3)
    held = torch.arange(tables.shape[1], device=tables.device) * BS < lens[:, None]
    return torch.where(held[:, None], x, -math.inf)


def _plain_select(s):
    c, x, lens = s["case"], s["scores"], s["seq_lens"].long()
    N, Hkv, width = x.shape
    at = torch.arange(width, device=x.device)
    held = ((lens + BS - 1) // BS)[:, None, None]
    x = torch.where((at < c["sink"]) | (at >= held - c["recent"]), math.inf, x)
    x = torch.where(at < held, x, math.nan)  # sorts behind everything below
    order = torch.sort(torch.nan_to_num(x, nan=-3e38, posinf=3e38, neginf=-2e38), dim=2, descending=True, stable=True).indices
    k = min(c["pages"], width)
    page = torch.where(order[:, :, :k] < held, order[:, :, :k], width).sort(2).values
    page = torch.where(page < width, page, -1)
    return torch.cat([page, page.new_full((N, Hkv, c["pages"] - k), -1)], 2).int()


def _plain_sparse(s):
    c, pages, lens = s["case"], s["pages"].long(), s["seq_lens"]
    N, Hkv, K = pages.shape
    D = c["dim"]
    n = torch.arange(N, device=pages.device)[:, None, None]
    block = s["tables"][n, pages.clamp(min=0)].long().clamp(min=0)
    head = torch.arange(Hkv, device=pages.device)[None, :, None]
    byte = torch.uint8 if c["kv"] == "fp8" else _TORCH[c["kv"]]
    k, v = [p.view(byte)[block, head].view(_TORCH[c["kv"]]).float().view(N, Hkv, K * BS, D) for p in (s["k_pool"], s["v_pool"])]
    if c["kv"] == "fp8":
        k, v = k * s["k_scales"][:, :, None, None], v * s["v_scales"][:, :, None, None]
    heads = _heads(c, pages.device)
    q = s["q"].float()[:, heads]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D)  # [N, Hkv, G, K * BS]
    pos = pages[..., None] * BS + torch.arange(BS, device=pages.device)
    seen = ((pages[..., None] >= 0) & (pos < lens[:, None, None, None])).view(N, Hkv, 1, K * BS)
    x = torch.where(seen, x, -math.inf)
    w = torch.exp(x - x.amax(3, keepdim=True).clamp(min=-3e38))
    o = torch.matmul(w, v) / w.sum(3, keepdim=True).clamp(min=1e-30)
    out = torch.empty_like(s["q"])
    out[:, heads] = o.to(out.dtype)
    return out


def run(s):
    if own:
        return _run_own(s)
    return {"tables": _plain_tables, "rope": _plain_rope, "bounds": _plain_bounds, "scores": _plain_scores, "select": _plain_select,
            "sparse": _plain_sparse}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "tables":
        before, new = _lens(case)
        granted = sum(_pages(b + n) - _pages(b) for b, n in zip(before, new))
        began = sum(1 for b, n in zip(before, new) if n and b % BS)  # tokens in a block that the table has
        rows = sum(new) + case["pad"]
        # lengths and offsets, granted blocks read and entered, entries read, a row's slot, position and sequence
        return {"bytes": len(new) * (4 + 4 + 4 + 8) + 8 * granted + 4 * began + 16 * rows, "flops": rows}
    Hkv = case["kv_heads"]
    if kind == "select":
        lens, _ = _lens(case)
        held = sum(_pages(n) for n in lens)
        return {"bytes": 4 * Hkv * (held + len(lens) * case["pages"]) + 4 * len(lens), "flops": Hkv * held}
    H, D = case["heads"], case["dim"]
    if kind == "rope":
        T, e = case["rows"], _BYTES[case["src"]]
        written = T * H * D * e + (T * Hkv * D * e if case["pool"] == "none" else 2 * T * Hkv * D * _BYTES[case["pool"]])
        read = T * (H + (1 if case["pool"] == "none" else 2) * Hkv) * D * e
        table = min(T, case["max_pos"]) * case["rot"] * 4
        return {"bytes": read + written + table + T * (4 if case["pool"] == "none" else 12),
                "flops": T * (H + Hkv) * (4 * D * case["norm"] + 3 * case["rot"])}
    if kind == "bounds":
        before, new = _lens(case)
        e = _BYTES[case["kv"]]
        pages = sum(_pages(b + n) - b // BS for b, n in zip(before, new))
        again = sum(1 for b in before if b % BS)  # begun pages, whose bounds are read too
        return {"bytes": sum(new) * (Hkv * D * e + 8) + 2 * Hkv * D * e * (pages + again), "flops": 2 * sum(new) * Hkv * D}
    lens, _ = _lens(case)
    held, e = sum(_pages(n) for n in lens), _BYTES[case["kv"]]
    rows = len(lens) * H * D * _BYTES[case["q"]]
    if kind == "scores":
        width = max(1, max(_pages(n) for n in lens))
        return {"bytes": held * (2 * Hkv * D * e + 4) + rows + 4 * len(lens) * (Hkv * width + 1), "flops": 4 * held * H * D}
    # selected tokens: at most `pages` pages of a sequence, the last of them as far as it is filled
    taken = sum(min(n, case["pages"] * BS - (-n) % BS) if case["pages"] > 1 else min(n, BS) for n in lens)
    listed_pages = sum(min(_pages(n), case["pages"]) for n in lens)
    return {"bytes": 2 * taken * Hkv * D * e + 2 * rows + Hkv * (4 * len(lens) * case["pages"] + 4 * listed_pages) + 4 * len(lens),
            "flops": 4 * taken * H * D}


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _exact_select(s):
    """Row by row on the host: the sorted list of the best pages, ties to the lower page."""
    import numpy as np

    c = s["case"]
    x, lens = s["scores"].double().cpu().numpy(), s["seq_lens"].cpu().numpy()
    N, Hkv, _ = x.shape
    out = np.full((N, Hkv, c["pages"]), -1, np.int32)
    for n in range(N):
        held = -(-int(lens[n]) // BS)
        for h in range(Hkv):
            row = x[n, h, :held].copy()
            row[:c["sink"]] = np.inf
            row[max(0, held - c["recent"]):] = np.inf
            best = np.lexsort((np.arange(held), -row))[:c["pages"]]
            out[n, h, :len(best)] = np.sort(best)
    return torch.from_numpy(out)


def _exact_tables(s):
    """Sequence by sequence on the host."""
    c = s["case"]
    before, new = _lens(c)
    tables, granted = s["tables"].cpu().clone(), s["blocks"].cpu().tolist()
    slots, positions, rows, cu, used = [], [], [], [0], 0
    for i, (b, n) in enumerate(zip(before, new)):
        row = tables[i].tolist()
        for p in range(_pages(b), _pages(b + n)):
            row[p] = granted[used]
            used += 1
        tables[i] = torch.tensor(row, dtype=torch.int32)
        for pos in range(b, b + n):
            slots.append(row[pos // BS] * BS + pos % BS)
            positions.append(pos)
            rows.append(i)
        cu.append(cu[-1] + n)
    pad = [-1] * c["pad"]
    return {"tables": tables, "slots": torch.tensor(slots + pad), "positions": torch.tensor(positions + pad, dtype=torch.int32),
            "rows": torch.tensor(rows + pad, dtype=torch.int32), "cu": torch.tensor(cu),
            "lens": torch.tensor([b + n for b, n in zip(before, new)], dtype=torch.int32), "cursor": torch.tensor([used])}


def _exact_rope(s):
    """Pairs as complex numbers: a rotation is a product with cos + i sin."""
    c = s["case"]
    T, H, Hkv, D, half = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["rot"] // 2
    x = s["qkv"].double().view(T, H + 2 * Hkv, D)
    turn = torch.complex(*s["rope"].double()[s["positions"].long()].split(half, 1))[:, None]

    def turned(x, w):
        if w is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        if c["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * half].reshape(T, -1, half, 2).contiguous()) * turn
            y = torch.view_as_real(z).reshape(T, -1, 2 * half)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        return torch.cat([y, x[..., 2 * half:]], -1)

    q, k, v = turned(x[:, :H], s["wq"]), turned(x[:, H:H + Hkv], s["wk"]), x[:, H + Hkv:]
    if c["pool"] == "none":
        return {"q": q, "k": k}
    pools = [torch.zeros(s["k_pool"].shape, dtype=torch.float64, device=q.device) for _ in range(2)]
    for pool, x, name in zip(pools, (k, v), ("k_scales", "v_scales")):
        if c["pool"] == "fp8":
            x = (x / s[name].double()[s["token_row"].long()][:, :, None]).clamp(-448, 448)
        flat = torch.zeros((pool.shape[0] * BS, Hkv, D), dtype=torch.float64, device=q.device)
        flat[s["slots"]] = x
        pool.copy_(flat.view(pool.shape[0], BS, Hkv, D).transpose(1, 2))
    return {"q": q, "k_pool": pools[0], "v_pool": pools[1]}


def _exact_bounds(s):
    """Token after token of each touched page on the host's side of the definition: a page that begins starts afresh."""
    out = s["bounds"].double()
    pool, slots = s["k_pool"].double(), s["slots"]
    for tib in range(BS):  # a page's tokens in their order
        block = slots[slots % BS == tib] // BS
        row = pool[block, :, tib]
        lo, hi = out[block, :, 0], out[block, :, 1]
        out[block, :, 0] = row if tib == 0 else torch.minimum(lo, row)
        out[block, :, 1] = row if tib == 0 else torch.maximum(hi, row)
    return out


def _exact_scores(s):
    c = s["case"]
    heads = _heads(c, "cuda")
    out = torch.full((c["seqs"], c["kv_heads"], s["tables"].shape[1]), -math.inf, dtype=torch.float64, device="cuda")
    lens, _ = _lens(c)
    for n, tokens in enumerate(lens):
        p = _pages(tokens)
        if p:
            b = s["bounds"][s["tables"][n, :p].long()].double()  # [p, Hkv, 2, D]
            for g in range(heads.shape[1]):
                q = s["q"][n, heads[:, g]].double()  # [Hkv, D]
                x = torch.maximum(q * b[:, :, 0], q * b[:, :, 1]).sum(2).t()
                out[n, :, :p] = torch.maximum(out[n, :, :p], x)
    return out


def _exact_sparse(s):
    c = s["case"]
    heads = _heads(c, "cuda")
    out = torch.zeros((c["seqs"], c["heads"], c["dim"]), dtype=torch.float64, device="cuda")
    lens, _ = _lens(c)
    for n, tokens in enumerate(lens):
        pages = s["pages"][n].long()  # [Hkv, K]
        pos = (pages[:, :, None] * BS + torch.arange(BS, device="cuda")).flatten(1)
        seen = (pages[:, :, None].expand(-1, -1, BS).flatten(1) >= 0) & (pos < tokens)
        if not tokens:
            continue
        block = s["tables"][n][pages.clamp(min=0)].long()
        head = torch.arange(c["kv_heads"], device="cuda")[:, None]
        k, v = [p.view(torch.uint8)[block, head].view(p.dtype).double().flatten(1, 2) if c["kv"] == "fp8" else p[block, head].double().flatten(1, 2)
                for p in (s["k_pool"], s["v_pool"])]
        if c["kv"] == "fp8":
            k, v = k * s["k_scales"][n].double()[:, None, None], v * s["v_scales"][n].double()[:, None, None]
        x = (s["q"][n][heads].double() @ k.transpose(1, 2)) / c["dim"] ** 0.5
        w = torch.softmax(torch.where(seen[:, None], x, -math.inf), 2)
        out[n, heads] = w @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "rope": _exact_rope, "bounds": _exact_bounds, "scores": _exact_scores, "select": _exact_select,
            "sparse": _exact_sparse}[case["kind"]](s)
