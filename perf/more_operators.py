"""Performance cases of the operators around a step's projections in 8 bits and with low-rank adapters: what a layer calls
between its attention and the next, for a model whose weights are kept in 8 bits and whose requests bring adapters of
their own.

A case is a dict of plain values; `kind` names the operator:

  norm    dense.rms_norm_fp8: the residual's addition and the root-mean-square norm, rows out in 8 bits with a scale each
  silu    dense.silu_mul_fp8: SiLU(gate) * up, out the same way
  linear  dense.linear_fp8: the product of such rows with a weight in 8 bits that has a scale a row
  plan    dense.lora_plan: a step's rows grouped by the adapter of their request
  lora    dense.lora: the rows' own low-rank products added to a shared projection's output

8 bits are e4m3 (largest value 448).  A row y is held as its scale s = max(max |y| / 448, 2^-126) and y / s rounded.
Every size belongs to the case, the values to the seed.  4096 columns,
32 / 8 heads of 128 (a fused projection of 4096 + 1024 + 1024 columns) and 14336 columns between gate and down are the
model shape of the repository's benchmark, 256 sequences its decode batch and 64 chunks of 512 its prefill batch.
"""
import math
import random

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f32": 4, "fp8": 1}
EPS = 1e-6
TOP = 448.0        # e4m3's largest value
LEAST = 2.0 ** -126  # smallest scale of a row


def listed():
    return [
        # one request's token between two layers
        dict(name="norm_token", kind="norm", rows=1, dim=4096, dtype="bf16", residual=True, select=0),
        # the decode batch's
        dict(name="norm_decode", kind="norm", rows=256, dim=4096, dtype="bf16", residual=True, select=0),
        # the prefill batch's
        dict(name="norm_chunks", kind="norm", rows=32768, dim=4096, dtype="bf16", residual=True, select=0),
        # gate and up of the decode batch, the halves of one projection's output
        dict(name="silu_decode", kind="silu", rows=256, cols=14336, dtype="bf16", fused=True),
        # those of 16 chunks of 512
        dict(name="silu_chunks", kind="silu", rows=8192, cols=14336, dtype="bf16", fused=True),
        # the down projection of one request's token: the weight is all there is to read
        dict(name="linear_token", kind="linear", m=1, n=4096, k=14336, out="bf16"),
        # gate and up for 64 decoding requests
        dict(name="linear_decode", kind="linear", m=64, n=28672, k=4096, out="bf16"),
        # the same for 16 chunks of 512
        dict(name="linear_chunks", kind="linear", m=8192, n=28672, k=4096, out="bf16"),
        # a decode step of 256 requests with 64 adapters among them, some without one
        dict(name="plan_decode", kind="plan", rows=256, adapters=64, run=1, without=0.2),
        # a prefill step: chunks of 512 rows, each of its request's adapter
        dict(name="plan_chunks", kind="plan", rows=32768, adapters=500, run=512, without=0.2),
        # query, key and value columns of 64 decoding requests with 32 adapters of rank 16
        dict(name="lora_decode", kind="lora", rows=64, adapters=32, rank=16, k=4096, cols="4096,1024,1024", x="bf16", dtype="bf16", run=1,
             without=0.1, ids_seed=1),
        # the attention's output projection of 16 chunks of 512 with 8 adapters of rank 32
        dict(name="lora_chunks", kind="lora", rows=8192, adapters=8, rank=32, k=4096, cols="4096", x="bf16", dtype="bf16", run=512,
             without=0.1, ids_seed=2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "silu", "linear", "linear", "lora", "lora", "plan"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "norm":
        dim = rng.choice([4096, 2048, 8192, 64, 16 * _log_int(rng, 4, 1000), _log_int(rng, 64, 4000)])
        rows = _log_int(rng, 1, max(2, min(16000, 60000000 // dim)))
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype, residual=rng.choice([True, True, False]),
                    select=rng.choice([0, 0, max(1, rows // 3)]))
    if kind == "silu":
        cols = rng.choice([14336, 4096, 11008, 16 * _log_int(rng, 4, 1000), _log_int(rng, 64, 4000)])
        return dict(kind=kind, rows=_log_int(rng, 1, max(2, min(8000, 50000000 // cols))), cols=cols, dtype=dtype, fused=rng.choice([True, False]))
    if kind == "linear":
        n, k = rng.choice([(4096, 4096), (6144, 4096), (28672, 4096), (4096, 14336), (_log_int(rng, 64, 16384), 16 * _log_int(rng, 4, 600)),
                           (_log_int(rng, 64, 16384), 16 * _log_int(rng, 4, 600))])
        return dict(kind=kind, m=_log_int(rng, 1, 4096), n=n, k=k, out=rng.choice(["bf16", "bf16", "f32"]))
    run = rng.choice([1, 1, 37, 512])
    if kind == "plan":
        return dict(kind=kind, rows=_log_int(rng, 1, 32768), adapters=_log_int(rng, 1, 2000), run=run, without=rng.choice([0.0, 0.2, 0.9]))
    rank = rng.choice([8, 16, 32, 64, _log_int(rng, 1, 128)])
    k, cols = rng.choice([(4096, "4096,1024,1024"), (4096, "14336,14336"), (14336, "4096"), (4096, "4096"),
                          (8 * _log_int(rng, 8, 500), str(_log_int(rng, 32, 4000)))])
    width = sum(_cols(cols))
    adapters = _log_int(rng, 1, max(2, min(64, 30000000 // (rank * (width + k)))))
    rows = _log_int(rng, 1, max(2, min(4096, 20000000 // width)))
    return dict(kind=kind, rows=rows, adapters=adapters, rank=rank, k=k, cols=cols, x=dtype if dtype == "f32" else rng.choice(["bf16", "bf16", "fp8"]),
                dtype=dtype, run=run, without=rng.choice([0.0, 0.2]), ids_seed=rng.randrange(1 << 20))


# ------------------------------------------------------------------ sizes and values

def _cols(text):
    return [int(w) for w in text.split(",")]


def _ids(case, seed=0):
    """Each row's adapter, in runs of `run` rows of one request; -1: none.  (A plan's are of the seed; a product's are of the
    case: they say which adapters it has to read.)"""
    rng = random.Random(seed if case["kind"] == "plan" else case["ids_seed"])
    out = []
    while len(out) < case["rows"]:
        a = -1 if rng.random() < case["without"] else rng.randrange(case["adapters"])
        out += [a] * (1 if case["run"] == 1 else rng.randint(1, case["run"]))
    return out[:case["rows"]]


def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed(seed * 64 + tag)


def _normal(seed, tag, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=_gen(seed, tag), device="cuda", dtype=torch.bfloat16 if dtype != "f32" else torch.float32)
    return (x * scale).to(_TORCH[dtype])


def _channels(seed, tag, n):
    """Sizes of a hidden state's columns: most alike, some a few times larger."""
    return 1 + 6 * (torch.rand(n, generator=_gen(seed, tag), device="cuda") < 0.01)


def _in_8_bits(y):
    """(rows in e4m3, scales) of f32 rows."""
    s = (y.abs().amax(1) / TOP).clamp(min=LEAST)
    return (y / s[:, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if kind == "norm":
        dt = case["dtype"]
        n, dim = (case["rows"] + case["select"], case["dim"])
        size = _channels(seed, 1, dim)
        s["x"] = (_normal(seed, 2, (n, dim), dt) * size).to(_TORCH[dt])
        s["residual"] = (_normal(seed, 3, (n, dim), dt) * size).to(_TORCH[dt]) if case["residual"] else None
        s["weight"] = (1 + _normal(seed, 4, (dim,), "f32", 0.1)).to(_TORCH[dt])
        # some rows of a step, as the last ones of its sequences
        s["rows"] = torch.randperm(n, generator=_gen(seed, 5), device="cuda")[:case["rows"]].sort().values if case["select"] else None
        return s
    if kind == "silu":
        gu = _normal(seed, 2, (case["rows"], 2 * case["cols"]), case["dtype"])
        s["gate"], s["up"] = gu[:, :case["cols"]], gu[:, case["cols"]:]
        if not case["fused"]:
            s["gate"], s["up"] = s["gate"].contiguous(), s["up"].contiguous()
        return s
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["x_scales"] = _in_8_bits((_normal(seed, 2, (m, k), "bf16") * _channels(seed, 3, k)).float())
        s["w"], s["w_scales"] = _in_8_bits(_normal(seed, 4, (n, k), "bf16", k ** -0.5).float())
        if own:  # laid out once, as a program does with a model's weights
            from zealot_amd import dense

            s["weight"] = dense.fp8_weight(s["w"], s["w_scales"])
        return s
    s["ids"] = torch.tensor(_ids(case, seed), dtype=torch.int32, device="cuda")
    if kind == "plan":
        return s
    dt, cols, r, A, k = case["dtype"], _cols(case["cols"]), case["rank"], case["adapters"], case["k"]
    x = _normal(seed, 2, (case["rows"], k), dt)
    s["x"], s["x_scales"] = _in_8_bits(x.float()) if case["x"] == "fp8" else (x, None)
    s["a"] = _normal(seed, 3, (A, len(cols) * r, k), dt, k ** -0.5)
    s["b"] = _normal(seed, 4, (A, sum(cols), r), dt, r ** -0.5)
    s["scales"] = 0.5 + torch.rand(A, generator=_gen(seed, 5), device="cuda")
    s["y"] = _normal(seed, 6, (case["rows"], sum(cols)), dt)
    if own:  # one of a step, for all its layers' projections
        from zealot_amd import dense

        s["plan"] = dense.lora_plan(s["ids"], A)
    return s


# ------------------------------------------------------------------ one pass

def _run_own(s):
    from zealot_amd import dense

    c, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        if s["residual"] is None:
            q = dense.rms_norm_fp8(s["x"], s["weight"], EPS, rows=s["rows"])
            return {"q": q.data, "scales": q.scales}
        q, t = dense.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["residual"], rows=s["rows"])
        return {"q": q.data, "scales": q.scales, "residual": t}
    if kind == "silu":
        q = dense.silu_mul_fp8(s["gate"], s["up"])
        return {"q": q.data, "scales": q.scales}
    if kind == "linear":
        return dense.linear_fp8(dense.Fp8Rows(s["x"], s["x_scales"]), s["weight"], out_dtype=_TORCH[c["out"]])
    if kind == "plan":
        p = dense.lora_plan(s["ids"], c["adapters"])
        return {"order": p.order, "offsets": p.offsets}
    x = s["x"] if s["x_scales"] is None else dense.Fp8Rows(s["x"], s["x_scales"])
    return dense.lora(x, s["a"], s["b"], s["scales"], s["plan"], s["y"], parts=tuple(_cols(c["cols"])))


def _plain_norm(s):
    x = s["x"] if s["rows"] is None else s["x"][s["rows"]]
    out = {}
    if s["residual"] is not None:
        x = (x.float() + (s["residual"] if s["rows"] is None else s["residual"][s["rows"]]).float()).to(x.dtype)
        out["residual"] = x
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["weight"].float()
    out["q"], out["scales"] = _in_8_bits(y)
    return out


def _plain_silu(s):
    g, u = s["gate"].float(), s["up"].float()
    q, scales = _in_8_bits(g / (1 + torch.exp(-g)) * u)
    return {"q": q, "scales": scales}


def _plain_linear(s):
    y = torch.matmul(s["x"].float(), s["w"].float().t())
    return (y * s["x_scales"][:, None] * s["w_scales"]).to(_TORCH[s["case"]["out"]])


def _plain_plan(s):
    A, ids = s["case"]["adapters"], s["ids"].long()
    key = torch.where((ids >= 0) & (ids < A), ids, A)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(A, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    order = torch.where(torch.arange(key.numel(), device=key.device) < offsets[-1], order, -1)
    return {"order": order.int(), "offsets": offsets.int()}


def _plain_lora(s):
    c, ids = s["case"], s["ids"].long()
    A, r, cols = c["adapters"], c["rank"], _cols(c["cols"])
    P, n = len(cols), sum(cols)
    x = s["x"].float()
    if s["x_scales"] is not None:
        x = x * s["x_scales"][:, None]
    # every row against every adapter, its own kept
    v = torch.matmul(x, s["a"].float().view(A * P * r, -1).t()).view(-1, A, P * r)
    v = v * ((ids[:, None] == torch.arange(A, device=ids.device)) * s["scales"])[:, :, None]
    # column j of part p meets the p-th r of an adapter's rows
    part = torch.repeat_interleave(torch.arange(P, device=ids.device), torch.tensor(cols, device=ids.device))
    w = s["b"].float().permute(0, 2, 1)[:, None] * (part == torch.arange(P, device=ids.device)[:, None])[None, :, None]
    s["y"].copy_(s["y"].float() + torch.matmul(v.view(-1, A * P * r), w.reshape(A * P * r, n)))
    return s["y"]


def run(s):
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "silu": _plain_silu, "linear": _plain_linear, "plan": _plain_plan, "lora": _plain_lora}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, dim, e = case["rows"], case["dim"], _BYTES[case["dtype"]]
        each = dim * (e * (3 if case["residual"] else 1) + 1) + 4 + (8 if case["select"] else 0)
        return {"bytes": n * each + dim * e, "flops": 6 * n * dim}
    if kind == "silu":
        n, cols, e = case["rows"], case["cols"], _BYTES[case["dtype"]]
        return {"bytes": n * (cols * (2 * e + 1) + 4), "flops": 7 * n * cols}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}
    ids = _ids(case)
    if kind == "plan":
        return {"bytes": 8 * len(ids) + 4 * (case["adapters"] + 1), "flops": len(ids)}
    e, cols, r, k = _BYTES[case["dtype"]], _cols(case["cols"]), case["rank"], case["k"]
    rows, used, n = sum(1 for a in ids if a >= 0), len({a for a in ids if a >= 0}), sum(cols)
    return {"bytes": max(1, rows * (k * _BYTES[case["x"]] + 2 * n * e + 8) + used * (r * e * (len(cols) * k + n) + 4)),
            "flops": 2 * rows * r * (len(cols) * k + n)}


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _exact_rows(y):
    """The 8-bit rows before their rounding, and their scales."""
    s = y.abs().max(dim=1).values / TOP
    return {"q": y / s.unsqueeze(1), "scales": s}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64
    if kind == "norm":
        t, kept = s["x"].to(f64), {}
        if case["residual"]:
            t = t + s["residual"].to(f64)
        if case["select"]:
            t = t.index_select(0, s["rows"])
        if case["residual"]:
            kept["residual"] = t
            t = t.to(_TORCH[case["dtype"]]).to(f64)  # the norm is of what the next layer reads
        y = t / (t.pow(2).sum(1) / case["dim"] + EPS).sqrt().unsqueeze(1) * s["weight"].to(f64)
        return {**_exact_rows(y), **kept}
    if kind == "silu":
        g = s["gate"].to(f64)
        return _exact_rows(torch.sigmoid(g) * g * s["up"].to(f64))
    if kind == "linear":
        x = s["x"].to(f64) * s["x_scales"].to(f64).unsqueeze(1)
        return x @ (s["w"].to(f64) * s["w_scales"].to(f64).unsqueeze(1)).T
    if kind == "plan":
        ids, A = _ids(case, seed), case["adapters"]
        lists = [[] for _ in range(A)]
        for i, a in enumerate(ids):
            if a >= 0:
                lists[a].append(i)
        flat, ends = [], [0]
        for rows in lists:
            flat += rows
            ends.append(len(flat))
        return {"order": torch.tensor(flat + [-1] * (len(ids) - len(flat)), dtype=torch.int32), "offsets": torch.tensor(ends, dtype=torch.int32)}
    ids = _ids(case)
    y, r, cols = s["y"].to(f64), case["rank"], _cols(case["cols"])
    for a in sorted(set(ids) - {-1}):
        rows = torch.tensor([i for i, b in enumerate(ids) if b == a], device="cuda")
        x = s["x"][rows].to(f64) if s["x_scales"] is None else s["x"].to(f64)[rows] * s["x_scales"][rows].to(f64).unsqueeze(1)
        first, delta = 0, []
        for p, width in enumerate(cols):
            low = x @ s["a"][a, p * r:(p + 1) * r].to(f64).T
            delta.append(low @ s["b"][a, first:first + width].to(f64).T)
            first += width
        y[rows] += float(s["scales"][a]) * torch.cat(delta, 1)
    return y
