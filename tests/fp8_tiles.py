"""What dense.linear_fp8 runs for a size: a restatement of the choice in
zealot_amd/csrc/fp8_gemm.hip (whose cost constants are read from there), and sizes
that reach every tile, with k whole and split.  Used by test_fp8_tiles.py (CPU) and
test_gpu_linear_fp8_tiles.py."""
import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zealot_amd", "csrc", "fp8_gemm.hip")


def _costs():
    with open(SOURCE) as f:
        text = f.read()
    names = re.search(r"enum \{ (k\d+x\d+(?:, k\d+x\d+)*), kTiles \};", text).group(1).replace("k", "").split(", ")
    rows = re.findall(r"\{(\d+), (\d+), ([\d.]+)f, ([\d.]+)f\}", text)
    assert len(rows) == len(names) == 9
    tiles = [(name, int(bm), int(bt), np.float32(a), np.float32(b)) for name, (bm, bt, a, b) in zip(names, rows)]
    assert all(name == f"{bm}x{16 * bt}" for name, bm, bt, _, _ in tiles)
    return tiles


TILES = _costs()


def choose(m: int, n: int, k: int, f32: bool):
    """(tile, splits of k, chunks a split) for more than 16 rows."""
    f = np.float32
    tiles, chunks = -(-n // 64) * 4, -(-k // 128)
    best, least = None, f(1e30)
    for name, bm, bt, start, chunk in TILES[:7] if f32 else TILES:
        big = name == "256x256"
        if big and chunks < 4:
            continue
        groups = -(-m // bm) * -(-tiles // bt)
        for s in (1,) if big else (1, 2, 4, 8):
            each = -(-chunks // s)
            if s > 1 and (each < 8 or groups * s > 512):
                break
            us = f((groups * s + 255) // 256) * (start + f(each) * chunk)
            if s > 1:
                us = us + (f(2.5) + f(s) * f(m) * f(tiles) * f(16) * f(8) / f(4e6))
            if us < least:
                least, best = us, (name, -(-chunks // each), each)
    return best


def stream(m: int, n: int) -> str:
    """The kernel of up to 16 rows: weight tiles a workgroup x waves."""
    tiles = -(-n // 64) * 4
    return "1x8" if tiles <= 256 else "1x4" if m <= 8 else "2x4" if tiles < 1024 else "4x4"


# (tile, splits, m, n, k): rows, columns and k that end inside tiles; split k: chunks that do
# not divide, an odd number of them a split for the tiles that take two at a time.
SIZES = {
    "bfloat16": [
        ("128x128", 1, 70, 16520, 528), ("128x128", 2, 65, 9243, 7712), ("128x128", 4, 66, 4433, 10064), ("128x128", 8, 65, 2147, 11808),
        ("128x64", 1, 2730, 648, 560), ("128x64", 2, 4183, 129, 13328), ("128x64", 4, 4253, 36, 7408), ("128x64", 8, 2161, 38, 9936),
        ("256x128", 1, 150, 22453, 544), ("256x128", 2, 129, 13115, 8784), ("256x128", 4, 145, 6281, 8880), ("256x128", 8, 213, 2087, 15136),
        ("256x256", 1, 340, 22666, 672), ("32x32", 1, 17, 40, 528), ("32x32", 4, 17, 33, 5200), ("32x32", 8, 20, 33, 8352),
        ("32x64", 1, 2184, 65, 560), ("32x64", 4, 17, 2049, 4272), ("32x64", 8, 17, 1054, 7408), ("64x128", 1, 19, 16890, 560),
        ("64x128", 2, 36, 8481, 8000), ("64x128", 4, 17, 4484, 9296), ("64x128", 8, 20, 2185, 9760), ("64x32", 1, 2102, 70, 816),
        ("64x32", 4, 33, 1106, 4192), ("64x32", 8, 296, 66, 8400), ("64x64", 1, 34, 8289, 528), ("64x64", 2, 265, 1585, 9312),
        ("64x64", 4, 1071, 67, 6176), ("64x64", 8, 1062, 33, 8560)],
    "float32": [
        ("128x128", 1, 69, 16863, 528), ("128x128", 2, 69, 8394, 8976), ("128x128", 4, 4152, 67, 9232), ("128x128", 8, 76, 2082, 10928),
        ("128x64", 1, 3384, 536, 528), ("128x64", 2, 4134, 137, 11312), ("128x64", 4, 4509, 34, 6496), ("128x64", 8, 2179, 33, 11600),
        ("32x32", 1, 18, 33, 544), ("32x32", 4, 17, 38, 4176), ("32x32", 8, 19, 34, 9008), ("32x64", 1, 17, 8293, 544),
        ("32x64", 4, 20, 2251, 4144), ("32x64", 8, 18, 1194, 7824), ("64x128", 1, 18, 16404, 528), ("64x128", 2, 34, 8810, 7264),
        ("64x128", 4, 18, 4236, 9312), ("64x128", 8, 17, 2349, 10848), ("64x32", 1, 4291, 33, 816), ("64x32", 4, 33, 1117, 4144),
        ("64x32", 8, 33, 541, 8496), ("64x64", 1, 33, 9087, 544), ("64x64", 2, 280, 1571, 10832), ("64x64", 4, 2149, 38, 5472),
        ("64x64", 8, 514, 68, 8656)],
}
TWO_CHUNKS = ("32x32", "64x32", "64x64")
