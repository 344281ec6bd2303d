"""Which tile and split a product in 8 bits takes (CPU): the restatement in fp8_tiles.py
against the library's own answers, and that the sizes of the GPU tests reach them all."""
import math
import random

import pytest

from tests.fp8_tiles import SIZES, TILES, TWO_CHUNKS, choose, stream
from zealot_amd import _lib

CODE = {"bfloat16": _lib.BF16, "float32": _lib.F32}


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_restatement_splits_as_the_library_does(dtype):
    rng = random.Random(2)
    for _ in range(4000):
        m, n, k = _log(rng, 17, 9000), _log(rng, 1, 33000), 16 * _log(rng, 1, 1100)
        splits = choose(m, n, k, dtype == "float32")[1]
        want = 0 if splits == 1 else splits * m * (-(-n // 64) * 64) * 4
        assert _lib.lib().zk_linear_fp8_workspace_size(m, n, k, CODE[dtype]) == want, (m, n, k)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_sizes_reach_every_tile_and_split(dtype):
    for tile, splits, m, n, k in SIZES[dtype]:
        got, s, each = choose(m, n, k, dtype == "float32")
        assert (got, s) == (tile, splits), (m, n, k, got, s)
        chunks = -(-k // 128)
        assert k % 128 and n % 64 and m % 16
        assert splits == 1 or chunks % each
        assert tile not in TWO_CHUNKS or each % 2
    # whatever else is chosen is one of these
    rng = random.Random(3)
    reached = {(tile, splits) for tile, splits, *_ in SIZES[dtype]}
    for _ in range(4000):
        size = _log(rng, 17, 9000), _log(rng, 1, 33000), 16 * _log(rng, 1, 1100)
        assert choose(*size, dtype == "float32")[:2] in reached, size
    assert {t for t, _ in reached} == {t[0] for t in (TILES[:7] if dtype == "float32" else TILES)}


def test_streams():
    assert [stream(*s) for s in ((9, 4096), (8, 5000), (9, 5000), (16, 16384), (9, 16321), (16, 28672))] == ["1x8", "1x4", "2x4", "4x4", "4x4", "4x4"]
