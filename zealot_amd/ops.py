"""Stateless torch-facing entry points of the paged-KV path.

Each function validates tensor shapes, dtypes and devices on the host and then
calls one C ABI entry point (include/zealot_kv.h) on torch's current stream.
Pools are 4-D tensors [num_blocks, Hkv, block_size, D] -- the layout of
src/kv_cache.rs:41-50 -- of dtype float32, bfloat16 or float8_e4m3fn (uint8
storage is accepted for fp8).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib

_ZK_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.uint8: _lib.FP8_E4M3}
if hasattr(torch, "float8_e4m3fn"):
    _ZK_DTYPES[torch.float8_e4m3fn] = _lib.FP8_E4M3


def zk_dtype(t: torch.Tensor) -> int:
    code = _ZK_DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return code


# The current stream's handle without the torch.cuda.Stream object around it:
# 0.2 us against 2.9, in calls whose launch takes 3.7 (a one-token append: 9.9 us
# of host time before, 5.5 with this and the checks below).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_get_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream(stream=None) -> int:
    """The address of `stream`, by default torch's current stream."""
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None or _get_device is None or not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_get_device())


def _dev(t: torch.Tensor, name: str, dtype=None, contiguous=True) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU (got {t.device})")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    return t.data_ptr()


def _opt(t, name, dtype=None):
    return None if t is None else _dev(t, name, dtype)


# Operands of the calls below _need: one expression a tensor on the way through
# (0.5 us; a fused norm + rotation + append names 14 of them), the reasons apart.

def _target(stream=None):
    """(torch's current device, which a launch goes to; the address of its stream, or of `stream`, which belongs to it)."""
    if stream is None and _raw_stream is not None and _get_device is not None and torch.cuda.is_initialized():
        cur = _get_device()
        return cur, _raw_stream(cur)
    if not torch.cuda.is_available():
        return -2, None  # (-1 is a host tensor's device: every operand is refused)
    cur = torch.cuda.current_device()
    if stream is not None and stream.device_index != cur:
        raise ValueError(f"stream is on device {stream.device_index}, the current device is {cur}")
    return cur, _stream(stream)


def _refuse(t, name: str, shape, dtype, cur: int):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU (got {t.device})")
    if t.get_device() != cur:
        raise ValueError(f"{name} is on {t.device}, the current device is {cur}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _need(t, name: str, shape, dtype, cur: int) -> int:
    """The address of a contiguous operand of this shape and type (None: any) on the current device."""
    try:
        ok = t.get_device() == cur and (dtype is None or t.dtype is dtype) and t.shape == shape and t.is_contiguous()
    except AttributeError:
        ok = False
    if not ok:
        _refuse(t, name, shape, dtype, cur)
    return t.data_ptr()


def _need_opt(t, name: str, shape, dtype, cur: int):
    return None if t is None else _need(t, name, shape, dtype, cur)


def _rows(t, name: str, rows: int, heads: int, dim: int, dtype, cur: int) -> int:
    """Elements from one token's row of an operand [rows, heads, dim] to the
    next: rows may lie apart (columns of a fused projection), a row is packed."""
    shape = (rows, heads, dim)
    try:
        ok = t.get_device() == cur and t.dtype is dtype and t.shape == shape
    except AttributeError:
        ok = False
    if not ok:
        _refuse(t, name, shape, dtype, cur)
    st = t.stride()
    if rows and ((st[2] != 1 and dim > 1) or (st[1] != dim and heads > 1) or (st[0] < heads * dim and rows > 1)):
        raise ValueError(f"{name} must have packed [heads, dim] rows that do not overlap")
    return st[0] if rows > 1 else heads * dim


def _dims(t, name: str, dims: str):
    """The shape of an operand of as many dimensions as `dims` names."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    shape = t.shape
    if len(shape) != dims.count(",") + 1:
        raise ValueError(f"{name} must be {dims}, got {list(shape)}")
    return shape


def _empty(like: torch.Tensor, shape, dtype, stream=None) -> torch.Tensor:
    """A new tensor for a launch on `stream`: the allocator reuses its memory in that stream's order."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _pool_shape(k_pool: torch.Tensor, v_pool: torch.Tensor):
    shape = k_pool.shape
    if len(shape) != 4 or shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool/v_pool must be equal 4-D tensors [num_blocks, Hkv, block_size, D]")
    return shape


def append(k_pool, v_pool, k, v, slot_mapping, k_scales=None, v_scales=None, token_row=None,
           stream=None) -> None:
    """Scatter k, v ([T, Hkv, D]) into the pools at slot_mapping[t] (int64)."""
    nb, hkv, bs, d = _pool_shape(k_pool, v_pool)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1] != hkv or k.shape[2] != d:
        raise ValueError(f"k/v must be [T, {hkv}, {d}], got {tuple(k.shape)} / {tuple(v.shape)}")
    if slot_mapping.shape != (k.shape[0],):
        raise ValueError("slot_mapping must be [T]")
    _lib.check(_lib.lib().zk_append(
        _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool"), zk_dtype(k_pool), _dev(k, "k"),
        _dev(v, "v"), zk_dtype(k), _dev(slot_mapping, "slot_mapping", torch.int64), k.shape[0],
        hkv, d, bs, nb, _opt(k_scales, "k_scales", torch.float32),
        _opt(v_scales, "v_scales", torch.float32), _opt(token_row, "token_row", torch.int32),
        _stream(stream)))


def fp8_scales(x, cu_seqlens, stream=None) -> torch.Tensor:
    """Per-(sequence, kv_head) scales amax/448 over x[cu[n]:cu[n+1]] ([T, Hkv, D])."""
    n = cu_seqlens.shape[0] - 1
    tokens, hkv, d = x.shape[0], x.shape[1], x.shape[2]
    out = torch.empty((n, hkv), dtype=torch.float32, device=x.device)
    # Parts of at least 64 tokens on average, up to two workgroups a CU, from 192 KB
    # a sequence and head on: below, the second launch and the scratch cost more
    # than the parts give (a call in parts is 11.7 us, most of it the host's; 8
    # heads of 128 bf16 undivided: 8 x 512 tokens 6.5 us, 8 x 1000 9.5, 8 x 2000 16.7).
    # (Not on a stream of the caller's choice: the scratch belongs to the current one.)
    split = stream is None and tokens * d * x.element_size() >= max(1, n) * (192 << 10)
    parts = min(512 // max(1, n * hkv), tokens // (64 * max(1, n))) if split else 1
    scratch = torch.empty(parts * n * hkv, dtype=torch.float32, device=x.device) if parts > 1 else None
    _lib.check(_lib.lib().zk_fp8_scales_parts(
        _dev(x, "x"), zk_dtype(x), _dev(cu_seqlens, "cu_seqlens", torch.int64), n, hkv, d, out.data_ptr(),
        scratch.data_ptr() if parts > 1 else None, max(1, parts), _stream(stream)))
    return out


def gather(k_pool, v_pool, block_tables, ctx_lens, out_offsets, k_out, v_out, stream=None) -> None:
    """Copy each sequence's first ctx_lens[n] tokens into rows out_offsets[n].. of k_out/v_out."""
    nb, hkv, bs, d = _pool_shape(k_pool, v_pool)
    n, mb = block_tables.shape
    if k_out.dtype != k_pool.dtype or v_out.dtype != k_pool.dtype:
        raise TypeError("gather outputs must have the pool dtype")
    _lib.check(_lib.lib().zk_gather(
        _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool"), zk_dtype(k_pool),
        _dev(block_tables, "block_tables", torch.int32), mb, _dev(ctx_lens, "ctx_lens", torch.int32),
        _dev(out_offsets, "out_offsets", torch.int64), n, _dev(k_out, "k_out"),
        _dev(v_out, "v_out"), hkv, d, bs, nb, _stream(stream)))


def copy_blocks(pools, src, dst, stream=None) -> None:
    """For each i: block dst[i] := block src[i] in every pool of `pools`."""
    if not pools:
        return
    shape = tuple(pools[0].shape)
    for p in pools:
        if tuple(p.shape) != shape or p.dtype != pools[0].dtype:
            raise ValueError("all pools must share shape and dtype")
    nb = shape[0]
    block_bytes = pools[0][0].numel() * pools[0].element_size()
    arr = (ctypes.c_void_p * len(pools))(*[_dev(p, "pool") for p in pools])
    if src.shape != dst.shape:
        raise ValueError("src and dst must have the same length")
    _lib.check(_lib.lib().zk_copy_blocks(
        arr, len(pools), block_bytes, nb, _dev(src, "src", torch.int32), _dev(dst, "dst", torch.int32),
        src.shape[0], _stream(stream)))


_MAPPINGS = {"grouped": _lib.GQA_GROUPED, "modulo": _lib.GQA_MODULO}


def decode_workspace_bytes(num_seqs, num_heads, head_dim, max_blocks_per_seq, block_size) -> int:
    return int(_lib.lib().zk_paged_decode_workspace_size(num_seqs, num_heads, head_dim,
                                                          max_blocks_per_seq, block_size))


def paged_decode(q, k_pool, v_pool, block_tables, seq_lens, scale=None, mapping="grouped",
                 k_scales=None, v_scales=None, out=None, workspace=None, stream=None):
    """Decode attention: q [N, H, D] (f32/bf16) over paged K/V; returns out [N, H, D]."""
    nb, hkv, bs, d = _pool_shape(k_pool, v_pool)
    if q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"q must be [N, H, {d}]")
    n, h, _ = q.shape
    if block_tables.dim() != 2 or block_tables.shape[0] != n or seq_lens.shape != (n,):
        raise ValueError("block_tables must be [N, max_blocks] and seq_lens [N]")
    mb = block_tables.shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)  # attention/cuda.rs:141
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must match q")
    if workspace is None:  # (one that is given is checked by the call)
        workspace = torch.empty(decode_workspace_bytes(n, h, d, mb, bs), dtype=torch.uint8, device=q.device)
    _lib.check(_lib.lib().zk_paged_decode(
        _dev(q, "q"), zk_dtype(q), _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool"),
        zk_dtype(k_pool), _dev(out, "out"), _dev(block_tables, "block_tables", torch.int32),
        _dev(seq_lens, "seq_lens", torch.int32), n, h, hkv, d, bs, mb, nb, float(scale),
        _MAPPINGS[mapping], _opt(k_scales, "k_scales", torch.float32),
        _opt(v_scales, "v_scales", torch.float32), _dev(workspace, "workspace"),
        workspace.numel() * workspace.element_size(), _stream(stream)))
    return out


class StepTables(NamedTuple):
    """What step_tables gives: rows are the step's tokens packed in batch order."""
    slot_mapping: torch.Tensor  # int64 [num_rows]; -1: no block, or no token
    positions: torch.Tensor     # int32 [num_rows]; -1: no token
    token_row: torch.Tensor     # int32 [num_rows], the token's sequence; -1: no token
    cu_seqlens: torch.Tensor    # int64 [N + 1]
    kv_lens: torch.Tensor       # int32 [N], lengths after the step
    cursor: torch.Tensor        # int64 [1], behind the granted blocks that the step takes


def step_tables(block_tables, seq_lens, new_lens, block_size: int, num_rows: int, new_blocks=None, cursor=None, out=None,
                stream=None) -> StepTables:
    """Block tables, slots and offsets of a step from its request lengths, on the
    GPU (zk_step_tables): sequence i holds seq_lens[i] tokens and receives
    new_lens[i] (int32 [N]); blocks it lacks are taken from new_blocks (int32,
    in batch order from cursor on, int64 [1]) and entered in block_tables (int32
    [N, max_blocks], in place).  num_rows: rows of the batch, padding included.
    out: a StepTables to write to; none of it may overlap an input."""
    n, mb = _dims(block_tables, "block_tables", "[N, max_blocks]")
    cur, at_stream = _target(stream)
    i32, i64 = torch.int32, torch.int64
    tables = _need(block_tables, "block_tables", (n, mb), i32, cur)
    lens, new = _need(seq_lens, "seq_lens", (n,), i32, cur), _need(new_lens, "new_lens", (n,), i32, cur)
    at = _need_opt(cursor, "cursor", (1,), i64, cur)
    granted, blocks = 0, None
    if new_blocks is not None:
        granted, = _dims(new_blocks, "new_blocks", "[blocks]")
        blocks = _need(new_blocks, "new_blocks", (granted,), i32, cur)
        if granted == 0:  # none were granted (a NULL list would mean that none are needed)
            blocks = tables
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    if out is None:  # one buffer a type
        # (the views are of memory that nothing else names)
        wide = _empty(block_tables, num_rows + n + 2, i64, stream)
        narrow = _empty(block_tables, 2 * num_rows + n, i32, stream)
        slots, cu, end = wide.unsafe_split_with_sizes((num_rows, n + 1, 1))
        pos, row, kv = narrow.unsafe_split_with_sizes((num_rows, num_rows, n))
        out = StepTables(slots, pos, row, cu, kv, end)
        p_slots, p_pos = wide.data_ptr(), narrow.data_ptr()
        p_cu, p_end = p_slots + 8 * num_rows, p_slots + 8 * (num_rows + n + 1)
        p_row, p_kv = p_pos + 4 * num_rows, p_pos + 8 * num_rows
    else:
        p_slots = _need(out.slot_mapping, "out.slot_mapping", (num_rows,), i64, cur)
        p_pos, p_row = [_need(t, name, (num_rows,), i32, cur)
                        for t, name in ((out.positions, "out.positions"), (out.token_row, "out.token_row"))]
        p_cu, p_kv = _need(out.cu_seqlens, "out.cu_seqlens", (n + 1,), i64, cur), _need(out.kv_lens, "out.kv_lens", (n,), i32, cur)
        p_end = _need(out.cursor, "out.cursor", (1,), i64, cur)
    _lib.check(_lib.lib().zk_step_tables(tables, n, mb, lens, new, block_size, blocks, granted, at, p_end, p_slots, p_pos,
                                         p_row, num_rows, p_cu, p_kv, at_stream))
    return out


_FLOAT = (torch.float32, torch.bfloat16)


def _rope_operands(positions, rope, q_weight, k_weight, tokens: int, dim: int, dtype, cur: int):
    """What both rope calls take besides q, k and v: ((weights), (positions, table, its rows, rot_dim))."""
    weights = (_need_opt(q_weight, "q_weight", (dim,), dtype, cur), _need_opt(k_weight, "k_weight", (dim,), dtype, cur))
    if rope is None:
        return weights, (None, None, 0, 0)
    most, rot = _dims(rope, "rope", "[max_positions, rot_dim]")
    if rot % 2 or rot > dim or rot == 0 or most == 0:
        raise ValueError(f"rope must be [max_positions, rot_dim] with an even rot_dim of at most {dim}")
    return weights, (_need(positions, "positions", (tokens,), torch.int32, cur),
                     _need(rope, "rope", (most, rot), torch.float32, cur), most, rot)


def qk_norm_rope_append(k_pool, v_pool, q, k, v, positions, slot_mapping, rope, q_weight=None, k_weight=None,
                        eps: float = 1e-6, interleaved: bool = False, q_out=None, k_scales=None, v_scales=None,
                        token_row=None, stream=None):
    """dense.qk_norm_rope of q [T, H, D] and k [T, Hkv, D], and append of the
    resulting K rows and of v at slot_mapping, in one launch: returns q_out
    (which may be q).  q, k and v may be columns of one fused projection output;
    K is rounded once, to the pool's type."""
    nb, hkv, bs, d = pool = _dims(k_pool, "k_pool", "[num_blocks, Hkv, block_size, D]")
    t, h, _ = _dims(q, "q", "[T, H, D]")
    dt = q.dtype
    if dt not in _FLOAT:
        raise TypeError(f"q must be float32 or bfloat16, got {dt}")
    cur, at_stream = _target(stream)
    qs, ks, vs = _rows(q, "q", t, h, d, dt, cur), _rows(k, "k", t, hkv, d, dt, cur), _rows(v, "v", t, hkv, d, dt, cur)
    if q_out is None:
        q_out, os_ = _empty(q, (t, h, d), dt, stream), 0
    else:
        os_ = _rows(q_out, "q_out", t, h, d, dt, cur)
    weights, table = _rope_operands(positions, rope, q_weight, k_weight, t, d, dt, cur)
    scales = (None, None, None)
    if k_scales is not None or v_scales is not None or token_row is not None:
        seqs, _ = _dims(k_scales, "k_scales", "[sequences, Hkv]")
        scales = (_need(k_scales, "k_scales", (seqs, hkv), torch.float32, cur),
                  _need(v_scales, "v_scales", (seqs, hkv), torch.float32, cur),
                  _need(token_row, "token_row", (t,), torch.int32, cur))
    kind = k_pool.dtype
    _lib.check(_lib.lib().zk_qk_norm_rope_append(
        _need(k_pool, "k_pool", pool, kind, cur), _need(v_pool, "v_pool", pool, kind, cur), zk_dtype(k_pool), q.data_ptr(),
        qs, k.data_ptr(), ks, v.data_ptr(), vs, _ZK_DTYPES[dt], t, h, hkv, d, *weights, eps, *table, interleaved,
        q_out.data_ptr(), os_, _need(slot_mapping, "slot_mapping", (t,), torch.int64, cur), bs, nb, *scales,
        at_stream))
    return q_out


def page_bounds(k_pool, slot_mapping, bounds, stream=None) -> None:
    """Bring the pages' key bounds ([num_blocks, Hkv, 2, D]: smallest, then
    largest, of the pool's type) up to date behind a write of K at slot_mapping
    (int64 [T]); the rows of one page are consecutive (zk_page_bounds)."""
    nb, hkv, bs, d = pool = _dims(k_pool, "k_pool", "[num_blocks, Hkv, block_size, D]")
    rows, = _dims(slot_mapping, "slot_mapping", "[T]")
    cur, at_stream = _target(stream)
    kind = k_pool.dtype
    _lib.check(_lib.lib().zk_page_bounds(
        _need(k_pool, "k_pool", pool, kind, cur), zk_dtype(k_pool),
        _need(slot_mapping, "slot_mapping", (rows,), torch.int64, cur), rows, hkv, d, bs, nb,
        _need(bounds, "bounds", (nb, hkv, 2, d), kind, cur), at_stream))


def page_scores(q, bounds, block_tables, seq_lens, block_size: int, mapping="grouped", out=None, stream=None):
    """An upper bound of q . k over each page's keys and the heads of a kv-head
    (zk_page_scores): q [N, H, D], scores f32 [N, Hkv, max_blocks], -inf behind
    the length."""
    shape = _dims(bounds, "bounds", "[num_blocks, Hkv, 2, D]")
    nb, hkv, two, d = shape
    if two != 2:
        raise ValueError("bounds must be [num_blocks, Hkv, 2, D]")
    n, h, _ = _dims(q, "q", "[N, H, D]")
    _, mb = _dims(block_tables, "block_tables", "[N, max_blocks]")
    cur, at_stream = _target(stream)
    if out is None:
        out = _empty(q, (n, hkv, mb), torch.float32, stream)
        scores = out.data_ptr()
    else:
        scores = _need(out, "out", (n, hkv, mb), torch.float32, cur)
    _lib.check(_lib.lib().zk_page_scores(
        _need(q, "q", (n, h, d), None, cur), zk_dtype(q), _need(bounds, "bounds", shape, None, cur), zk_dtype(bounds),
        _need(block_tables, "block_tables", (n, mb), torch.int32, cur), _need(seq_lens, "seq_lens", (n,), torch.int32, cur),
        scores, n, h, hkv, d, block_size, mb, nb, _MAPPINGS[mapping], at_stream))
    return out


def select_pages(scores, seq_lens, block_size: int, num_pages: int, sink: int = 1, recent: int = 1, out=None, stream=None):
    """The num_pages best pages of each (sequence, kv-head) in ascending order
    (int32 [N, Hkv, num_pages], then -1), the first `sink` and last `recent` held
    ones always among them; equal scores: the lower page (zk_select_pages)."""
    n, hkv, mb = shape = _dims(scores, "scores", "[N, Hkv, max_blocks]")
    if num_pages <= 0:
        raise ValueError("num_pages must be positive")
    cur, at_stream = _target(stream)
    if out is None:
        out = _empty(scores, (n, hkv, num_pages), torch.int32, stream)
        pages = out.data_ptr()
    else:
        pages = _need(out, "out", (n, hkv, num_pages), torch.int32, cur)
    _lib.check(_lib.lib().zk_select_pages(
        _need(scores, "scores", shape, torch.float32, cur), _need(seq_lens, "seq_lens", (n,), torch.int32, cur), n, hkv, mb,
        block_size, num_pages, sink, recent, pages, at_stream))
    return out


def sparse_workspace_bytes(num_seqs, num_heads, num_kv_heads, head_dim, num_pages) -> int:
    return int(_lib.lib().zk_paged_decode_sparse_workspace_size(num_seqs, num_heads, num_kv_heads, head_dim, num_pages))


def paged_decode_sparse(q, k_pool, v_pool, block_tables, seq_lens, pages, scale=None, mapping="grouped", k_scales=None,
                        v_scales=None, out=None, workspace=None, stream=None):
    """paged_decode over listed pages only: pages int32 [N, Hkv, K] holds indices
    into each sequence's block table (negative: none), as select_pages gives
    them; returns out [N, H, D] (zk_paged_decode_sparse)."""
    nb, hkv, bs, d = pool = _dims(k_pool, "k_pool", "[num_blocks, Hkv, block_size, D]")
    n, h, _ = _dims(q, "q", "[N, H, D]")
    _, mb = _dims(block_tables, "block_tables", "[N, max_blocks]")
    _, _, np_ = _dims(pages, "pages", "[N, Hkv, num_pages]")
    cur, at_stream = _target(stream)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dt = q.dtype
    if out is None:
        out = _empty(q, (n, h, d), dt, stream)
        dst = out.data_ptr()
    else:
        dst = _need(out, "out", (n, h, d), dt, cur)
    need = _lib.lib().zk_paged_decode_sparse_workspace_size(n, h, hkv, d, np_) if workspace is None else 0
    if need:
        workspace = _empty(q, need, torch.uint8, stream)
    ws = (None, 0)
    if workspace is not None:  # (its size is checked by the call)
        ws = (_need(workspace, "workspace", workspace.shape, None, cur), workspace.numel() * workspace.element_size())
    kind = k_pool.dtype
    _lib.check(_lib.lib().zk_paged_decode_sparse(
        _need(q, "q", (n, h, d), dt, cur), zk_dtype(q), _need(k_pool, "k_pool", pool, kind, cur),
        _need(v_pool, "v_pool", pool, kind, cur), zk_dtype(k_pool), dst,
        _need(block_tables, "block_tables", (n, mb), torch.int32, cur), _need(seq_lens, "seq_lens", (n,), torch.int32, cur),
        _need(pages, "pages", (n, hkv, np_), torch.int32, cur), np_, n, h, hkv, d, bs, mb, nb, scale, _MAPPINGS[mapping],
        _need_opt(k_scales, "k_scales", (n, hkv), torch.float32, cur),
        _need_opt(v_scales, "v_scales", (n, hkv), torch.float32, cur), *ws, at_stream))
    return out


def prefill_workspace_bytes(num_seqs, total_q, num_heads, num_kv_heads) -> int:
    return int(_lib.lib().zk_paged_prefill_workspace_size(num_seqs, total_q, num_heads, num_kv_heads))


def paged_prefill(q, k_pool, v_pool, block_tables, cu_seqlens_q, start_pos, causal=True, scale=None,
                  mapping="grouped", k_scales=None, v_scales=None, out=None, workspace=None, stream=None):
    """Chunked-prefill attention: q [T, H, D] (f32/bf16), sequence n's chunk is
    rows cu_seqlens_q[n] .. cu_seqlens_q[n+1] (int64) after start_pos[n] (int32)
    cached tokens; its K/V must already be in the pages.  Returns out [T, H, D]."""
    nb, hkv, bs, d = _pool_shape(k_pool, v_pool)
    if q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"q must be [T, H, {d}]")
    t, h, _ = q.shape
    n = start_pos.shape[0]
    if block_tables.dim() != 2 or block_tables.shape[0] != n or cu_seqlens_q.shape != (n + 1,):
        raise ValueError("block_tables must be [N, max_blocks], cu_seqlens_q [N + 1] and start_pos [N]")
    mb = block_tables.shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must match q")
    if workspace is None:
        workspace = torch.empty(prefill_workspace_bytes(n, t, h, hkv), dtype=torch.uint8, device=q.device)
    _lib.check(_lib.lib().zk_paged_prefill(
        _dev(q, "q"), zk_dtype(q), _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool"), zk_dtype(k_pool),
        _dev(out, "out"), _dev(block_tables, "block_tables", torch.int32),
        _dev(cu_seqlens_q, "cu_seqlens_q", torch.int64), _dev(start_pos, "start_pos", torch.int32), n, t, h, hkv,
        d, bs, mb, nb, float(scale), int(bool(causal)), _MAPPINGS[mapping],
        _opt(k_scales, "k_scales", torch.float32), _opt(v_scales, "v_scales", torch.float32),
        _dev(workspace, "workspace"), workspace.numel() * workspace.element_size(), _stream(stream)))
    return out
