"""The rules that the 8-bit products' kernels go by, without a GPU: which bytes a
load of a tile's rows may read, and which kernel the sizes of the GPU tests take."""
import ctypes

import pytest

import f8_rules
import test_gpu_f8
import test_gpu_f8_gated
from test_gpu_f8_tiles import GATED, TILES


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    return f8_rules.build(tmp_path_factory.mktemp("f8"))


def readable(nbytes, scalar, at):
    """Whether a lane at `at` reads memory: the range check of a raw buffer, which takes the scalar offset from the bytes
    in unsigned arithmetic."""
    return at < (nbytes - scalar) % 2 ** 32


@pytest.mark.parametrize("most", [16, 32, 64])  # rows of one load: of a stream's wave, of four and eight waves of a tile
@pytest.mark.parametrize("rows,pitch", [(1, 128), (7, 256), (33, 640), (200, 384), (2 ** 12, 2 ** 21)])
def test_loads_stay_in_the_matrix(rules, most, rows, pitch):
    """Rows that are there are read whole, at their column block, and what lies past the matrix's end is not: for loads
    partly and wholly behind it, and for a workgroup past its last tile (none left, wherever it stands)."""
    last, to = pitch // 128 - 1, (ctypes.c_int * 2)()
    for first in sorted({0, 1, most - 1, most, max(rows - most, 0), max(rows - 1, 0), rows, rows + 1, rows + 255}):
        for left in {rows - first, min(rows - first, 0) - 5, min(rows - first, 0)}:
            rules.rule_piece(first, left, rows, most, to)
            base, nbytes = to[0], to[1] * pitch
            assert 0 <= base and base + to[1] <= rows
            assert left < 1 or base == first
            for block in {0, last // 2, last}:
                for row in range(most):
                    for column in (0, 16, 112):
                        at = row * pitch + column
                        if readable(nbytes, block * 128, at):
                            assert base * pitch + block * 128 + at + 16 <= rows * pitch
                            assert row < max(left, 1)
                        else:
                            assert row >= left
    assert readable(0, 128, 0)  # what a scalar offset does to a buffer of no rows


@pytest.mark.parametrize("type,tokens,cols,rows,tile_tokens,tile_rows,tiles,steps", TILES + GATED)
def test_sizes_take_their_tiles(rules, type, tokens, cols, rows, tile_tokens, tile_rows, tiles, steps):
    w = f8_rules.way(rules, type, tokens, cols, rows)
    assert w.persistent and (w.tokens, w.rows, w.tiles, w.steps) == (tile_tokens, tile_rows, tiles, steps), w


def test_every_kernel_has_sizes(rules):
    """Every shape of the tables is taken by a GPU test's size: shares of the columns by its lists of them, tiles by one
    step, by several tiles of an even number of steps and by several of an odd one."""
    to = (ctypes.c_int * 4)()
    known = {"f32": 9, "bf16": 10, "hidden": 4}
    tiles = {(c[0],) + c[4:6] for c in TILES + GATED}
    streams = set()
    for s in test_gpu_f8.SHAPES + test_gpu_f8.STREAMS + test_gpu_f8_gated.SIZES:
        for type in ("f32", "bf16", "gated"):
            w = f8_rules.way(rules, type, *s)
            if not w.persistent:
                streams.add((w.kind, w.tokens, w.rows))
    for type, count in known.items():
        for i in range(count):
            rules.rule_listed(f8_rules.OUT[type], i, to)
            assert to[0] > 0
            shape = (type, to[0], to[1])
            assert shape in (streams if to[3] > 1 else tiles), shape
        if count < 10:
            rules.rule_listed(f8_rules.OUT[type], count, to)
            assert to[0] == 0
    for t in tiles | {("gated", 128, 128), ("gated", 256, 128)}:
        runs = {(c[6] > 1, c[7] == 1, c[7] % 2) for c in TILES + GATED if (c[0],) + c[4:6] == t}
        assert {(True, False, 0), (True, False, 1)} <= runs, t
        # f32 tiles of 256 x 128 are chosen from fourteen steps on
        assert (False, True, 1) in runs or t == ("f32", 256, 128), t


def test_gated_sizes(rules):
    ways = [f8_rules.way(rules, "gated", *s) for s in test_gpu_f8_gated.SIZES]
    assert [(w.tokens, w.rows) for w in ways] == [(16, 16), (32, 16), (128, 128), (256, 128)], ways
