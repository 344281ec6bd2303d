"""Dense ops around the paged-KV path over the C ABI (include/zealot_dense.h):
rms_norm (optionally fused with the residual add), silu_mul, add, embedding,
qk_norm_rope (head norms and rotary embedding) and linear (hipBLASLt or the weight-streaming kernel; TiledWeight for weights
kept in that kernel's tiled layout); rms_norm_fp8, silu_mul_fp8 and linear_fp8
(rows and weights in 8 bits); lora_plan and lora (low-rank adapters of the
requests beside a shared projection).  Torch device tensors in, launches on
torch's current stream; the kernels are in zealot_amd/csrc/dense_ops.hip,
rope_ops.hip, gemm.cpp, skinny_gemm.hip, fp8_rows.hip, fp8_gemm.hip and lora_ops.hip."""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from .ops import _dev, _dims, _empty, _need, _need_opt, _rope_operands, _rows, _stream, _target, zk_dtype


def _dt(t: torch.Tensor) -> int:
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"dense ops take float32 or bfloat16 tensors, got {t.dtype}")
    return zk_dtype(t)


def _sized(t, name: str, numel: int, dtype) -> None:
    """The kernels take plain pointers and trust the sizes: every operand is
    checked against the elements and dtype the launch will touch."""
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} elements, the op needs {numel}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def rms_norm(x, weight, eps: float = 1e-6, residual=None, out=None, residual_out=None, rows=None, stream=None):
    """out = rms_norm(s) * weight, s = x (+ residual, written to residual_out,
    which may be `residual`), over x's rows or over the rows listed in `rows`
    (device int64); rms_norm.cu:4-55."""
    dim = x.shape[-1]
    n = rows.numel() if rows is not None else x.numel() // dim
    if rows is None and x.numel() != n * dim:
        raise ValueError("x must hold whole rows of dim elements")
    if out is None:
        out = torch.empty((n, dim), dtype=x.dtype, device=x.device)
    if residual is not None and residual_out is None:
        residual_out = torch.empty((n, dim), dtype=x.dtype, device=x.device)
    _sized(weight, "weight", dim, x.dtype)
    _sized(out, "out", n * dim, x.dtype)
    if rows is None:
        _sized(residual, "residual", n * dim, x.dtype)
    elif residual is not None and (residual.numel() != x.numel() or residual.dtype != x.dtype):
        raise ValueError("residual must match x (its rows are selected by `rows` too)")
    _sized(residual_out, "residual_out", n * dim, x.dtype)
    _lib.check(_lib.lib().zk_rms_norm(
        _dev(x, "x"), None if residual is None else _dev(residual, "residual"), _dev(weight, "weight"),
        _dev(out, "out"), None if residual_out is None else _dev(residual_out, "residual_out"),
        None if rows is None else _dev(rows, "rows", torch.int64), n, dim, float(eps), _dt(x), _stream(stream)))
    return out if residual is None else (out, residual_out)


def silu_mul(gate, up, out=None, stream=None):
    """silu(gate) * up (activation.cu:4-12); gate / up may be column slices
    of one [rows, 2 * cols] tensor (a fused gate|up projection)."""
    rows, cols = gate.shape
    if up.dtype != gate.dtype:
        raise TypeError("gate and up must share a dtype")
    for name, t in (("gate", gate), ("up", up)):
        _dev(t, name, contiguous=False)
        if t.shape != (rows, cols) or t.stride(1) != 1:
            raise ValueError(f"{name} must be [rows, cols] with contiguous rows")
    if out is None:
        out = torch.empty((rows, cols), dtype=gate.dtype, device=gate.device)
    _sized(out, "out", rows * cols, gate.dtype)
    _lib.check(_lib.lib().zk_silu_mul(gate.data_ptr(), up.data_ptr(), _dev(out, "out"), rows, cols, gate.stride(0),
                                      up.stride(0), _dt(gate), _stream(stream)))
    return out


def add(a, b, out=None, stream=None):
    _sized(b, "b", a.numel(), a.dtype)
    if out is None:
        out = torch.empty_like(a)
    _sized(out, "out", a.numel(), a.dtype)
    _lib.check(_lib.lib().zk_add(_dev(a, "a"), _dev(b, "b"), _dev(out, "out"), a.numel(), _dt(a), _stream(stream)))
    return out


def embedding(ids, table, out=None, stream=None):
    """table[ids] (embedding.cu:4-22); out-of-range ids give zero rows."""
    n = ids.numel()
    if out is None:
        out = torch.empty((n, table.shape[1]), dtype=table.dtype, device=table.device)
    _sized(out, "out", n * table.shape[1], table.dtype)
    _lib.check(_lib.lib().zk_embedding(_dev(ids, "ids", torch.int64), _dev(table, "table"), _dev(out, "out"), n,
                                       table.shape[0], table.shape[1], _dt(table), _stream(stream)))
    return out


def rope_table(max_positions: int, rot_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """The position table of qk_norm_rope (f32 [max_positions, rot_dim]): row p
    holds cos(p theta^(-2 i / rot_dim)) for i < rot_dim / 2, then the sines.
    Angles are formed in 64 bits, so far positions keep their phase."""
    if max_positions <= 0 or rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rope_table needs positions and an even rot_dim")
    freq = float(theta) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def qk_norm_rope(q, k, positions, rope, q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None, stream=None):
    """RMSNorm of the query and key heads (q [T, H, D], k [T, Hkv, D]; weights
    [D], None: no norm) and the rotary embedding of their first rot_dim dimensions
    by the rows `positions` (int32 [T]) of `rope` (rope_table; None: no
    rotation) in one pass: returns (q_out, k_out).  q and k may be columns of a
    fused projection output, and q_out / k_out those columns themselves."""
    t, h, d = _dims(q, "q", "[T, H, D]")
    _, hkv, _ = _dims(k, "k", "[T, Hkv, D]")
    dt = q.dtype
    code = _dt(q)
    cur, at_stream = _target(stream)
    qs, ks = _rows(q, "q", t, h, d, dt, cur), _rows(k, "k", t, hkv, d, dt, cur)
    qo = ko = 0
    if q_out is None:
        q_out = _empty(q, (t, h, d), dt, stream)
    else:
        qo = _rows(q_out, "q_out", t, h, d, dt, cur)
    if k_out is None:
        k_out = _empty(k, (t, hkv, d), dt, stream)
    else:
        ko = _rows(k_out, "k_out", t, hkv, d, dt, cur)
    weights, table = _rope_operands(positions, rope, q_weight, k_weight, t, d, dt, cur)
    _lib.check(_lib.lib().zk_qk_norm_rope(
        q.data_ptr(), qs, k.data_ptr(), ks, code, t, h, hkv, d, *weights, eps, *table, interleaved, q_out.data_ptr(), qo,
        k_out.data_ptr(), ko, at_stream))
    return q_out, k_out


class TiledWeight:
    """A bf16 weight [n, k] in the weight-streaming kernel's tiled layout
    (zk_weight_tile): [k / 128][n / 16][16 rows][16 units of 8], unit u of row
    r holding columns 8 (u ^ r) .. of its 128-column chunk.  linear,
    linear_rms_norm and linear_silu_mul take it in place of the row-major
    tensor; the products read it with contiguous 1 KiB loads (17-19 % faster
    on the large decode projections).  `data` is the flat device buffer.

    The weight-streaming kernel reads the whole weight once per 64 rows of
    x, so it suits decode-sized products only.  `full`, when kept (the
    row-major [n, k] weight), serves products of more than TILED_MAX_ROWS
    rows (prefill and mixed steps) on zk_linear's GEMM plan instead."""

    __slots__ = ("data", "n", "k", "full")

    def __init__(self, data: torch.Tensor, n: int, k: int, full: torch.Tensor | None = None):
        if data.dtype != torch.bfloat16 or data.numel() != n * k or not data.is_contiguous():
            raise ValueError("a tiled weight is a contiguous bf16 buffer of n * k elements")
        if full is not None and (full.dtype != torch.bfloat16 or tuple(full.shape) != (n, k)
                                 or not full.is_contiguous()):
            raise ValueError("the row-major copy is a contiguous bf16 [n, k] tensor")
        self.data, self.n, self.k, self.full = data, n, k, full

    @property
    def shape(self):
        return (self.n, self.k)

    @property
    def dtype(self):
        return self.data.dtype

    @property
    def device(self):
        return self.data.device

    def numel(self) -> int:
        return self.n * self.k

    def rowmajor(self) -> torch.Tensor:
        """The row-major [n, k] weight (the inverse permutation, on the device)."""
        n, k = self.n, self.k
        # moved as int16 words, so every bit pattern (NaN payloads too) survives
        t = self.data.view(torch.int16).view(k // 128, n // 16, 16, 16, 8).permute(1, 2, 0, 3, 4)  # [b r j u e]
        r = torch.arange(16, device=t.device).view(16, 1)
        idx = (torch.arange(16, device=t.device).view(1, 16) ^ r).view(1, 16, 1, 16, 1).expand(t.shape)
        return torch.gather(t, 3, idx).reshape(n, k).view(torch.bfloat16)  # [b r j c e] = t[b r j (c ^ r) e]


def tile_weight(weight: torch.Tensor, stream=None, keep_full: bool = False) -> TiledWeight:
    """The tiled form of a row-major bf16 weight [n, k] (n % 16 == 0,
    k % 128 == 0), in a new buffer; keep_full keeps `weight` beside it for
    products of more than TILED_MAX_ROWS rows."""
    n, k = weight.shape
    if weight.dtype != torch.bfloat16:
        raise ValueError("tiled weights are bf16")
    out = torch.empty(n * k, dtype=torch.bfloat16, device=weight.device)
    _lib.check(_lib.lib().zk_weight_tile(_dev(weight, "weight"), _dev(out, "out"), n, k, _stream(stream)))
    return TiledWeight(out, n, k, weight.contiguous() if keep_full else None)


# Rows of x up to which a TiledWeight's product runs on the weight-streaming
# kernel even when its row-major copy is kept: that kernel reads the weight
# once per 64 rows, a GEMM once.
TILED_MAX_ROWS = 64


def _route(x, weight):
    """The weight a product of x runs on: a TiledWeight's row-major copy for
    more than TILED_MAX_ROWS rows, when it keeps one."""
    if isinstance(weight, TiledWeight) and weight.full is not None and x.shape[0] > TILED_MAX_ROWS:
        return weight.full
    return weight


def _tiled_x(x, weight):
    if x.dtype != torch.bfloat16 or x.shape[1] != weight.k:
        raise ValueError("tiled weights take bf16 x [m, k]")


def linear(x, weight, out=None, out_dtype=None, stream=None):
    """x [m, k] . weight[n, k]^T on hipBLASLt (the cublasSgemm_v2 sites) or the
    weight-streaming kernel, whichever the first call of the shape timed
    faster; a TiledWeight runs on the weight-streaming kernel (on its
    row-major copy, if kept, for more than TILED_MAX_ROWS rows)."""
    m, k = x.shape
    n = weight.shape[0]
    weight = _route(x, weight)
    if isinstance(weight, TiledWeight):
        _tiled_x(x, weight)
        if out is None:
            out = torch.empty((m, n), dtype=out_dtype or x.dtype, device=x.device)
        _sized(out, "out", m * n, out.dtype)  # the C ABI checks the dtype pair
        _lib.check(_lib.lib().zk_linear_tiled(_dev(x, "x"), _dev(weight.data, "weight"), _dev(out, "out"), m, n, k,
                                              zk_dtype(out), _stream(stream)))
        return out
    if weight.shape[1] != k or weight.dtype != x.dtype:
        raise ValueError("weight must be [n, k] of x's dtype")
    od = out_dtype or x.dtype
    if out is None:
        out = torch.empty((m, n), dtype=od, device=x.device)
    _sized(out, "out", m * n, out.dtype)  # the C ABI checks the dtype pair
    _lib.check(_lib.lib().zk_linear(_dev(x, "x"), _dev(weight, "weight"), _dev(out, "out"), m, n, k, _dt(x),
                                    zk_dtype(out), _stream(stream)))
    return out


def linear_rms_norm(x, weight, norm_weight, eps: float = 1e-6, residual=None, out=None, residual_out=None,
                    stream=None):
    """rms_norm(linear(x, weight), norm_weight, eps, residual, ...) bit for
    bit, for bf16 in two launches instead of three when the projection runs on
    the weight-streaming kernel with split k (its sums feed the norm
    directly); f32 runs the two calls.  Returns out, or (out, residual_out)
    with a residual."""
    m, k = x.shape
    n = weight.shape[0]
    if weight.shape[1] != k or weight.dtype != x.dtype:
        raise ValueError("weight must be [n, k] of x's dtype")
    weight = _route(x, weight)
    tiled = isinstance(weight, TiledWeight)
    if tiled:
        _tiled_x(x, weight)
    elif x.dtype != torch.bfloat16:
        return rms_norm(linear(x, weight), norm_weight, eps, residual=residual, out=out, residual_out=residual_out,
                        stream=stream)
    if out is None:
        out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    if residual is not None and residual_out is None:
        residual_out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    _sized(norm_weight, "norm_weight", n, x.dtype)
    for name, t in (("out", out), ("residual", residual), ("residual_out", residual_out)):
        _sized(t, name, m * n, x.dtype)
    fn = _lib.lib().zk_linear_rms_norm_tiled if tiled else _lib.lib().zk_linear_rms_norm
    _lib.check(fn(
        _dev(x, "x"), _dev(weight.data if tiled else weight, "weight"), m, n, k,
        None if residual is None else _dev(residual, "residual"),
        _dev(norm_weight, "norm_weight"), float(eps), _dev(out, "out"),
        None if residual_out is None else _dev(residual_out, "residual_out"), _stream(stream)))
    return out if residual is None else (out, residual_out)


GATE_UP_BLOCK = 16  # rows of gate (then of up) per block of a fused gate|up weight


def interleave_gate_up(gate, up):
    """The fused [2 I, hidden] gate|up weight for linear_silu_mul: gate and up
    rows interleaved in blocks of GATE_UP_BLOCK."""
    i, hid = gate.shape
    if up.shape != gate.shape or i % GATE_UP_BLOCK:
        raise ValueError("gate and up must be [I, hidden] with I a multiple of 16")
    b = GATE_UP_BLOCK
    return torch.stack([gate.reshape(i // b, b, hid), up.reshape(i // b, b, hid)], 1).reshape(2 * i, hid).contiguous()


def split_gate_up(gate_up):
    """(gate, up) of a weight from interleave_gate_up."""
    n, hid = gate_up.shape
    b = GATE_UP_BLOCK
    v = gate_up.reshape(n // (2 * b), 2, b, hid)
    return v[:, 0].reshape(n // 2, hid), v[:, 1].reshape(n // 2, hid)


def linear_silu_mul(x, gate_up, out=None, gu=None, stream=None):
    """silu(x . gate^T) * (x . up^T) for a gate|up weight from
    interleave_gate_up, bit for bit linear() followed by SiLU * up of its
    rounded outputs; for bf16 one launch when the projection runs on the
    weight-streaming kernel without split."""
    m, k = x.shape
    n = gate_up.shape[0]
    if gate_up.shape[1] != k or gate_up.dtype != x.dtype or n % (2 * GATE_UP_BLOCK):
        raise ValueError("gate_up must be [2 I, k] of x's dtype, I a multiple of 16")
    gate_up = _route(x, gate_up)
    if isinstance(gate_up, TiledWeight):  # one launch, no projection buffer
        _tiled_x(x, gate_up)
        if out is None:
            out = torch.empty((m, n // 2), dtype=x.dtype, device=x.device)
        _sized(out, "out", m * (n // 2), x.dtype)
        _lib.check(_lib.lib().zk_linear_silu_mul_tiled(_dev(x, "x"), _dev(gate_up.data, "gate_up"), _dev(out, "out"),
                                                       m, n // 2, k, _stream(stream)))
        return out
    if x.dtype != torch.bfloat16:  # f32: the projection, then SiLU * up of its column blocks
        y = linear(x, gate_up).view(m, n // (2 * GATE_UP_BLOCK), 2, GATE_UP_BLOCK)
        return silu_mul(y[:, :, 0].reshape(m, n // 2), y[:, :, 1].reshape(m, n // 2), out=out, stream=stream)
    if out is None:
        out = torch.empty((m, n // 2), dtype=x.dtype, device=x.device)
    if gu is None:
        gu = torch.empty((m, n), dtype=x.dtype, device=x.device)
    _sized(out, "out", m * (n // 2), x.dtype)
    _sized(gu, "gu", m * n, x.dtype)
    _lib.check(_lib.lib().zk_linear_silu_mul(_dev(x, "x"), _dev(gate_up, "gate_up"), _dev(out, "out"), m, n // 2, k,
                                             _dev(gu, "gu"), _stream(stream)))
    return out


# ------------------------------------------------------------------ projections in 8 bits

class Fp8Rows(NamedTuple):
    """Rows in 8 bits: e4m3 values [m, k] and one float32 scale a row [m]; a
    row's values are data * scale."""
    data: torch.Tensor
    scales: torch.Tensor


_FP8 = torch.float8_e4m3fn
FP8_LONGEST_ROW = 32768  # columns of bfloat16 rows that rms_norm_fp8 and silu_mul_fp8 write (whole vectors of 8)
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _fp8_out(out, like, rows: int, cols: int, cur: int, stream):
    """(the Fp8Rows to write, addresses of its values and scales)."""
    if out is None:
        out = Fp8Rows(_empty(like, (rows, cols), _FP8, stream), _empty(like, (rows,), torch.float32, stream))
        return out, out.data.data_ptr(), out.scales.data_ptr()
    return out, _need(out.data, "out.data", (rows, cols), _FP8, cur), _need(out.scales, "out.scales", (rows,), torch.float32, cur)


def rms_norm_fp8(x, weight, eps: float = 1e-6, residual=None, out=None, residual_out=None, rows=None, stream=None):
    """rms_norm with the rows written in 8 bits for linear_fp8
    (zk_rms_norm_fp8): returns Fp8Rows, or (Fp8Rows, residual_out) with a
    residual.  x [T, dim]; rows (device int64) selects some of them, one outside
    x gives zeros; residual_out may be x or `residual` when rows is None."""
    t, dim = _dims(x, "x", "[T, dim]")
    dt = x.dtype
    code = _dt(x)
    cur, at_stream = _target(stream)
    px, pw = _need(x, "x", (t, dim), dt, cur), _need(weight, "weight", (dim,), dt, cur)
    pr, n, pi = _need_opt(residual, "residual", (t, dim), dt, cur), t, None
    if rows is not None:
        n, = _dims(rows, "rows", "[rows]")
        pi = _need(rows, "rows", (n,), torch.int64, cur)
    po = None
    if residual is not None:
        if residual_out is None:
            residual_out = _empty(x, (n, dim), dt, stream)
            po = residual_out.data_ptr()
        else:
            po = _need(residual_out, "residual_out", (n, dim), dt, cur)
    out, pq, ps = _fp8_out(out, x, n, dim, cur, stream)
    # (an empty selection has no address: NULL would mean all rows)
    _lib.check(_lib.lib().zk_rms_norm_fp8(px, pr, pw, pq, ps, po, pi if n else px, t, n, dim, eps, code, at_stream))
    return out if residual is None else (out, residual_out)


def silu_mul_fp8(gate, up, out=None, stream=None):
    """silu_mul with the rows written in 8 bits for linear_fp8
    (zk_silu_mul_fp8): gate and up [rows, cols] may be column slices of one
    tensor; returns Fp8Rows."""
    rows, cols = _dims(gate, "gate", "[rows, cols]")
    dt = gate.dtype
    code = _dt(gate)
    cur, at_stream = _target(stream)
    gs, us = _rows2(gate, "gate", rows, cols, dt, cur), _rows2(up, "up", rows, cols, dt, cur)
    out, pq, ps = _fp8_out(out, gate, rows, cols, cur, stream)
    _lib.check(_lib.lib().zk_silu_mul_fp8(gate.data_ptr(), up.data_ptr(), pq, ps, rows, cols, gs, us, code, at_stream))
    return out


def _rows2(t, name: str, rows: int, cols: int, dtype, cur: int) -> int:
    """Elements from one row of an operand [rows, cols] to the next; a row is packed."""
    try:
        ok = t.get_device() == cur and t.dtype is dtype and t.shape == (rows, cols)
    except AttributeError:
        ok = False
    if not ok:
        _need(t, name, (rows, cols), dtype, cur)
    st = t.stride()
    if rows and ((st[1] != 1 and cols > 1) or (st[0] < cols and rows > 1)):
        raise ValueError(f"{name} must have packed rows that do not overlap")
    return st[0] if rows > 1 else cols


class Fp8Weight:
    """A weight [n, k] in 8 bits with one float32 scale a row (`scales` [n]), in
    the packed order that linear_fp8 reads (zk_fp8_weight; fp8_weight makes
    one).  `data` is the flat device buffer."""

    __slots__ = ("data", "scales", "n", "k")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, n: int, k: int):
        if data.dtype != torch.uint8 or data.dim() != 1 or data.numel() != _lib.lib().zk_fp8_weight_bytes(n, k) or not data.is_contiguous():
            raise ValueError("a packed weight is a flat uint8 buffer of zk_fp8_weight_bytes(n, k)")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (n,) or not scales.is_contiguous():
            raise ValueError("scales must be float32 [n]")
        if scales.device != data.device:
            raise ValueError("scales must be on the packed weight's device")
        self.data, self.scales, self.n, self.k = data, scales, n, k

    @property
    def shape(self):
        return (self.n, self.k)

    @property
    def device(self):
        return self.data.device

    def numel(self) -> int:
        return self.n * self.k

    def rowmajor(self) -> torch.Tensor:
        """The e4m3 values, row-major [n, k] (the inverse permutation, on the device)."""
        groups, chunks = -(-self.n // 64), -(-self.k // 128)
        # [G tile chunk unit 4 4 byte]: row 64 G + 16 i1 + 4 tile + i0, column 128 chunk + 16 unit + byte
        t = self.data.view(groups, 4, chunks, 8, 4, 4, 16).permute(0, 4, 1, 5, 2, 3, 6)
        return t.reshape(groups * 64, chunks * 128)[:self.n, :self.k].contiguous().view(_FP8)


def fp8_weight(weight: torch.Tensor, scales: torch.Tensor | None = None, stream=None) -> Fp8Weight:
    """The 8-bit packed form of a weight [n, k] (nn.Linear layout): float32 or
    bfloat16 values, rounded with a scale a row, or float8_e4m3fn values with
    their float32 `scales` [n]."""
    n, k = _dims(weight, "weight", "[n, k]")
    ready = weight.dtype == _FP8
    if not ready:
        _dt(weight)
    if ready != (scales is not None):
        raise ValueError("scales go with float8_e4m3fn weights")
    cur, at_stream = _target(stream)
    pw = _need(weight, "weight", (n, k), weight.dtype, cur)
    if n == 0 or k == 0:
        raise ValueError("weight must not be empty")
    if ready:
        _need(scales, "scales", (n,), torch.float32, cur)
    else:
        scales = _empty(weight, (n,), torch.float32, stream)
    data = _empty(weight, (_lib.lib().zk_fp8_weight_bytes(n, k),), torch.uint8, stream)
    _lib.check(_lib.lib().zk_fp8_weight(pw, zk_dtype(weight), data.data_ptr(), scales.data_ptr(), n, k, at_stream))
    return Fp8Weight(data, scales, n, k)


@functools.lru_cache(1024)
def _fp8_ws(m: int, n: int, k: int, code: int) -> int:
    return _lib.lib().zk_linear_fp8_workspace_size(m, n, k, code)


def linear_fp8_workspace_bytes(m: int, n: int, k: int, out_dtype=torch.bfloat16) -> int:
    return int(_lib.lib().zk_linear_fp8_workspace_size(m, n, k, _CODES[out_dtype]))


def linear_fp8(x: Fp8Rows, weight: Fp8Weight, out=None, out_dtype=torch.bfloat16, workspace=None, stream=None):
    """x . weight^T for rows and a weight in 8 bits (zk_linear_fp8): y [m, n],
    bfloat16 or float32 (`out_dtype`, or out's own).  k % 16 == 0."""
    if not isinstance(x, Fp8Rows):
        raise TypeError("x must be Fp8Rows (rms_norm_fp8 and silu_mul_fp8 give them)")
    m, k = _dims(x.data, "x.data", "[m, k]")
    if not isinstance(weight, Fp8Weight):
        raise TypeError("weight must be an Fp8Weight (fp8_weight makes one)")
    n = weight.n
    if weight.k != k:
        raise ValueError(f"x has {k} columns, the weight {weight.k}")
    cur, at_stream = _target(stream)
    px, ps = _need(x.data, "x.data", (m, k), _FP8, cur), _need(x.scales, "x.scales", (m,), torch.float32, cur)
    pw, pws = _need(weight.data, "weight", weight.data.shape, torch.uint8, cur), _need(weight.scales, "weight.scales", (n,), torch.float32, cur)
    if out is None:
        if out_dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"out_dtype must be float32 or bfloat16, got {out_dtype}")
        out = _empty(x.data, (m, n), out_dtype, stream)
        py = out.data_ptr()
    else:
        py = _need(out, "out", (m, n), None, cur)
        _dt(out)
    lib, code = _lib.lib(), zk_dtype(out)
    ws = (None, 0)
    if workspace is not None:  # (its size is checked by the call)
        ws = (_need(workspace, "workspace", workspace.shape, None, cur), workspace.numel() * workspace.element_size())
    elif m > 16:
        size = _fp8_ws(m, n, k, code)
        if size:
            workspace = _empty(out, (size,), torch.uint8, stream)  # (held until the launch is made)
            ws = (workspace.data_ptr(), size)
    _lib.check(lib.zk_linear_fp8(px, ps, pw, pws, py, m, n, k, code, *ws, at_stream))
    return out


# ------------------------------------------------------------------ low-rank adapters

class LoraPlan(NamedTuple):
    """A step's rows grouped by adapter (lora_plan), for all its projections."""
    order: torch.Tensor    # int32 [T]: the rows with an adapter, sorted by it; then -1
    offsets: torch.Tensor  # int32 [adapters + 1]: where each adapter's rows begin in it
    tiles: torch.Tensor    # int32 [tiles, 2]: the kernels' own


def lora_plan(adapter_ids, num_adapters: int, out: LoraPlan | None = None, stream=None) -> LoraPlan:
    """Group the rows of a step by adapter (zk_lora_plan): adapter_ids int32 [T],
    outside [0, num_adapters): none."""
    t, = _dims(adapter_ids, "adapter_ids", "[T]")
    cur, at_stream = _target(stream)
    i32 = torch.int32
    ids = _need(adapter_ids, "adapter_ids", (t,), i32, cur)
    if num_adapters <= 0:
        raise ValueError("num_adapters must be positive")
    tiles = _lora_tiles(t, num_adapters)
    if out is None:  # one buffer, the tiles first
        buf = _empty(adapter_ids, (2 * tiles + t + num_adapters + 1,), i32, stream)
        part = buf.split_with_sizes((2 * tiles, t, num_adapters + 1))
        out = LoraPlan(part[1], part[2], part[0].view(tiles, 2))
    _lib.check(_lib.lib().zk_lora_plan(ids, t, num_adapters, _need(out.order, "out.order", (t,), i32, cur),
                                       _need(out.offsets, "out.offsets", (num_adapters + 1,), i32, cur),
                                       _need(out.tiles, "out.tiles", (tiles, 2), i32, cur), at_stream))
    return out


# Sizes depend on a call's numbers alone: asked for once each (0.6 us a question, of a
# call's 10).
@functools.lru_cache(1024)
def _lora_tiles(rows: int, adapters: int) -> int:
    return _lib.lib().zk_lora_max_tiles(rows, adapters)


@functools.lru_cache(1024)
def _lora_sizes(rows: int, adapters: int, k: int, rank: int, parts: int, code: int):
    return _lora_tiles(rows, adapters), _lib.lib().zk_lora_workspace_size(rows, adapters, k, rank, parts, code)


@functools.lru_cache(1024)
def _columns(parts: tuple):
    return (ctypes.c_int64 * len(parts))(*parts), sum(parts)


def lora_workspace_bytes(num_rows: int, num_adapters: int, k: int, rank: int, num_parts: int, dtype) -> int:
    return int(_lib.lib().zk_lora_workspace_size(num_rows, num_adapters, k, rank, num_parts, _CODES[dtype]))


def lora(x, a, b, scales, plan: LoraPlan, y, parts=None, part_block: int = 0, workspace=None, stream=None):
    """y += scales[i] b[i] (a[i] x) row by row, i the row's adapter in `plan`
    (zk_lora; of as many adapters); rows without one stay as they are.  x [T, k] (rows may lie apart)
    of the weights' type, or Fp8Rows beside bfloat16 weights; a [adapters, P * rank,
    k], b [adapters, n, rank], scales float32 [adapters] or None; y [T, n], in
    place (rows may lie apart: columns of a fused output).  parts: the columns of
    y's P parts, each with ranks of its own (None: one), or, with part_block, how
    many parts take turns of part_block columns.  Returns y."""
    na, n, rank = _dims(b, "b", "[adapters, n, rank]")
    dt = b.dtype
    code = _dt(b)
    rows = x.data if isinstance(x, Fp8Rows) else x
    t, k = _dims(rows, "x", "[T, k]")
    cur, at_stream = _target(stream)
    cols, p = None, 1
    if part_block:
        if not isinstance(parts, int) or parts < 1:
            raise ValueError("with part_block, parts is their number")
        p = parts
    elif parts is not None:
        p = len(parts)
        cols, total = _columns(tuple(parts))
        if p == 0 or total != n:
            raise ValueError(f"parts must add up to the {n} columns of y")
    if plan.offsets.shape[0] != na + 1:  # (rows of an adapter that is not there would be left out without a word)
        raise ValueError(f"the plan is of {plan.offsets.shape[0] - 1} adapters, the weights of {na}")
    if isinstance(x, Fp8Rows):
        xc, xs = _lib.FP8_E4M3, _rows2(rows, "x.data", t, k, _FP8, cur)
        sc = _need(x.scales, "x.scales", (t,), torch.float32, cur)
    else:
        xc, xs, sc = code, _rows2(rows, "x", t, k, dt, cur), None
    ys = _rows2(y, "y", t, n, dt, cur)
    lib = _lib.lib()
    i32 = torch.int32
    tiles, size = _lora_sizes(t, na, k, rank, p, code)
    if workspace is None:
        workspace = _empty(y, (size,), torch.uint8, stream)  # (held until the launches are made)
        ws = (workspace.data_ptr() if size else None, size)
    else:
        ws = (_need(workspace, "workspace", workspace.shape, None, cur), workspace.numel() * workspace.element_size())
    _lib.check(lib.zk_lora(
        rows.data_ptr(), sc, xs, xc, _need(a, "a", (na, p * rank, k), dt, cur), _need(b, "b", (na, n, rank), dt, cur),
        _need_opt(scales, "scales", (na,), torch.float32, cur), code, _need(plan.order, "plan.order", (t,), i32, cur),
        _need(plan.tiles, "plan.tiles", (tiles, 2), i32, cur), t, na, k, n,
        rank, p, cols, part_block, y.data_ptr(), ys, *ws, at_stream))
    return y


def linear_choice(m, n, k, in_dtype=torch.bfloat16, out_dtype=None, tiled=False) -> dict:
    """What the projection plan for this shape runs (after a first call made
    it): splits 0 = hipBLASLt, else the weight-streaming kernel with that split
    of k and tile_rows; fused_* is what linear_rms_norm runs.  tiled: the plan
    for a TiledWeight of that shape."""
    import ctypes
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
    c = (ctypes.c_int * 4)()
    if tiled:
        _lib.check(_lib.lib().zk_linear_tiled_choice(m, n, k, code[out_dtype or in_dtype], c))
    else:
        _lib.check(_lib.lib().zk_linear_choice(m, n, k, code[in_dtype], code[out_dtype or in_dtype], c))
    return {"splits": c[0], "tile_rows": c[1], "fused_splits": c[2], "fused_rows": c[3]}


def pin_split(m, n, k, fused_splits, fused_rows, in_dtype=torch.bfloat16, out_dtype=None, tiled=False) -> None:
    """Pin the split-k configuration linear_rms_norm / write_batch_qkv fold
    for the plan an earlier call made for this shape (fused_splits 0: none)."""
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
    _lib.check(_lib.lib().zk_linear_pin_split(m, n, k, code[in_dtype], code[out_dtype or in_dtype], int(tiled),
                                              fused_splits, fused_rows))


def linear_skinny(x, weight, splits=1, tile_rows=128, out=None, out_dtype=None, stream=None):
    """The weight-streaming kernel zk_linear may choose for bf16 and m <= 64,
    called directly: tiles of tile_rows weight rows, k split in `splits`."""
    m, k = x.shape
    n = weight.shape[0]
    if weight.shape[1] != k or weight.dtype != torch.bfloat16 or x.dtype != torch.bfloat16:
        raise ValueError("x and weight must be bf16, weight [n, k]")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype or x.dtype, device=x.device)
    _lib.check(_lib.lib().zk_linear_skinny(_dev(x, "x"), _dev(weight, "weight"), _dev(out, "out"), m, n, k,
                                           zk_dtype(out), tile_rows, splits, _stream(stream)))
    return out
