"""ops.step_tables on the MI355X against a plain walk over the sequences: the
tables, slots, positions and offsets of a step from its request lengths, with
granted blocks and without, batches past one workgroup's threads, sequences
without tokens, padding, too few blocks, full tables; and a run of them: the
slots feed append and decode, and a captured call replays.  All results are
whole numbers, so they have to be equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _walk(tables, before, new, bs, num_rows, granted, cursor):
    """The definition, sequence by sequence."""
    tables = tables.copy()
    n, width = tables.shape
    cap = width * bs
    slots, pos, row, cu, lens = [], [], [], [0], []
    for i in range(n):
        s, t = max(int(before[i]), 0), max(int(new[i]), 0)
        if granted is not None:
            for p in range(-(-min(s, cap) // bs), -(-min(s + t, cap) // bs)):
                entry = granted[cursor] if cursor < len(granted) else -1
                if cu[-1] + p * bs - s < num_rows:  # the block's first token has a row
                    tables[i, p] = entry
                cursor += 1
        for x in range(s, s + t):
            b = tables[i, x // bs] if x < cap else -1
            slots.append(int(b) * bs + x % bs if b >= 0 else -1)
            pos.append(x)
            row.append(i)
        cu.append(cu[-1] + t)
        lens.append(min(s + t, cap))
    pad = max(0, num_rows - len(slots))
    return (tables, np.array(slots[:num_rows] + [-1] * pad, np.int64), np.array(pos[:num_rows] + [-1] * pad, np.int32),
            np.array(row[:num_rows] + [-1] * pad, np.int32), np.array(cu, np.int64), np.array(lens, np.int32), cursor)


def _case(rng, n, hi, new_hi, bs, slack=2):
    before = rng.integers(0, hi + 1, n).astype(np.int32)
    new = rng.integers(0, new_hi + 1, n).astype(np.int32)
    width = max(1, int(max((before + new + bs - 1) // bs)) + slack)
    pages = (before + bs - 1) // bs
    need = int(sum((before + new + bs - 1) // bs - pages))
    blocks = rng.permutation(int(pages.sum()) + need).astype(np.int32)
    tables = -np.ones((n, width), np.int32)
    o = 0
    for i in range(n):
        tables[i, :pages[i]] = blocks[o:o + pages[i]]
        o += pages[i]
    return tables, before, new, blocks[o:], int(new.sum())


def _call(tables, before, new, bs, num_rows, granted, cursor=None, **kw):
    from zealot_amd import ops
    dev = lambda a, t: None if a is None else torch.tensor(a, dtype=t, device="cuda")  # noqa: E731
    bt = dev(tables, torch.int32)
    out = ops.step_tables(bt, dev(before, torch.int32), dev(new, torch.int32), bs, num_rows, dev(granted, torch.int32),
                          dev(cursor, torch.int64), **kw)
    return bt, out


def _check(got, ref):
    bt, out = got
    tables, slots, pos, row, cu, lens, cursor = ref
    for a, b in ((bt, tables), (out.slot_mapping, slots), (out.positions, pos), (out.token_row, row), (out.cu_seqlens, cu),
                 (out.kv_lens, lens)):
        np.testing.assert_array_equal(a.cpu().numpy(), b)
    assert out.cursor.item() == cursor


@pytest.mark.parametrize("n,hi,new_hi,bs,pad", [(1, 0, 1, 16, 0), (1, 100, 40, 16, 3), (7, 50, 0, 16, 5), (64, 300, 200, 16, 0),
                                                (256, 900, 1, 16, 0), (257, 40, 5, 16, 9), (1000, 33, 3, 1, 0), (5000, 70, 2, 16, 1),
                                                (3, 1000, 700, 37, 2), (300, 5, 300, 64, 100)])
def test_against_the_walk(n, hi, new_hi, bs, pad):
    rng = np.random.default_rng(n * 31 + hi)
    tables, before, new, granted, total = _case(rng, n, hi, new_hi, bs)
    _check(_call(tables, before, new, bs, total + pad, granted), _walk(tables, before, new, bs, total + pad, granted, 0))


def test_tables_that_hold_every_block():
    rng = np.random.default_rng(2)
    tables, before, new, granted, total = _case(rng, 20, 100, 50, 16)
    full = _walk(tables, before, new, 16, total, granted, 0)[0]
    bt, out = _call(full, before, new, 16, total, None)
    ref = _walk(full, before, new, 16, total, None, 0)
    _check((bt, out), ref)


def test_a_cursor_goes_on_and_few_blocks_show():
    rng = np.random.default_rng(3)
    tables, before, new, granted, total = _case(rng, 20, 100, 50, 16)
    some = np.concatenate([np.full(5, 9999, np.int32), granted])
    _check(_call(tables, before, new, 16, total, some, [5]), _walk(tables, before, new, 16, total, some, 5))
    few = granted[:len(granted) // 2]
    bt, out = _call(tables, before, new, 16, total, few)
    ref = _walk(tables, before, new, 16, total, few, 0)
    _check((bt, out), ref)
    assert out.cursor.item() > len(few) and (out.slot_mapping == -1).any()
    _check(_call(tables, before, new, 16, total, granted[:0]), _walk(tables, before, new, 16, total, granted[:0], 0))


def test_full_tables_and_lengths_below_zero():
    rng = np.random.default_rng(4)
    tables = rng.integers(0, 50, (4, 3)).astype(np.int32)
    before, new = np.array([40, 48, 60, -5], np.int32), np.array([20, 3, 1, 7], np.int32)  # the table holds 48
    granted = np.arange(100, 110, dtype=np.int32)
    total = int(new.sum())
    _check(_call(tables, before, new, 16, total, granted), _walk(tables, before, new, 16, total, granted, 0))
    new[0] = -3
    _check(_call(tables, before, new, 16, 11, granted), _walk(tables, before, new, 16, 11, granted, 0))


def test_fewer_rows_than_tokens():
    rng = np.random.default_rng(5)
    tables, before, new, granted, total = _case(rng, 9, 60, 40, 16)
    rows = total // 2
    _check(_call(tables, before, new, 16, rows, granted), _walk(tables, before, new, 16, rows, granted, 0))


def test_entries_of_other_pages_stay():
    """Only the new tokens' blocks are written, whatever stands elsewhere in the table."""
    rng = np.random.default_rng(6)
    tables, before, new, granted, total = _case(rng, 30, 100, 40, 16, slack=5)
    tables[tables < 0] = 777
    bt, _ = _call(tables, before, new, 16, total, granted)
    want = _walk(tables, before, new, 16, total, granted, 0)[0]
    np.testing.assert_array_equal(bt.cpu().numpy(), want)


def test_empty_batch():
    bt, out = _call(np.zeros((0, 4), np.int32), np.zeros(0, np.int32), np.zeros(0, np.int32), 16, 3, None, [4])
    assert out.cu_seqlens.tolist() == [0] and out.cursor.item() == 4 and out.slot_mapping.tolist() == [-1] * 3


def test_captured_steps_of_a_decode_loop():
    """One captured call advances a batch token by token: lengths and cursor are
    copied back between the replays, other eager work runs among them."""
    from zealot_amd import ops
    rng = np.random.default_rng(7)
    n, bs, steps = 40, 16, 40
    before = rng.integers(0, 50, n).astype(np.int32)
    tables = -np.ones((n, 8), np.int32)
    pages = (before + bs - 1) // bs
    ids = rng.permutation(int(pages.sum()) + n * 4).astype(np.int32)
    o = 0
    for i in range(n):
        tables[i, :pages[i]] = ids[o:o + pages[i]]
        o += pages[i]
    granted = ids[o:]
    bt, lens = torch.tensor(tables, device="cuda"), torch.tensor(before, device="cuda")
    new, blocks = torch.ones(n, dtype=torch.int32, device="cuda"), torch.tensor(granted, device="cuda")
    cursor = torch.zeros(1, dtype=torch.int64, device="cuda")
    out = ops.step_tables(bt.clone(), lens, new, bs, n, blocks, cursor)  # warm
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.step_tables(bt, lens, new, bs, n, blocks, cursor, out=out)
    host, length, at = tables, before.copy(), 0
    for _ in range(steps):
        g.replay()
        ref = _walk(host, length, np.ones(n, np.int32), bs, n, granted, at)
        _check((bt, out), ref)
        host, length, at = ref[0], ref[5], ref[6]
        lens.copy_(out.kv_lens)
        cursor.copy_(out.cursor)
        torch.ones(1000, device="cuda").sum()
        torch.cuda.synchronize()


def test_another_stream():
    rng = np.random.default_rng(8)
    tables, before, new, granted, total = _case(rng, 64, 300, 200, 16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    got = _call(tables, before, new, 16, total, granted, stream=s)
    s.synchronize()
    _check(got, _walk(tables, before, new, 16, total, granted, 0))
