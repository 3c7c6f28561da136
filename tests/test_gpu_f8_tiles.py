"""Every persistent tile of the 8-bit products on the GPU, over one tile a workgroup and several, with odd and even
numbers of steps (a workgroup's next tile then begins in the other buffer of LDS, or in the same), against sums that
are exact in f32. tests/test_f8_rules.py holds the sizes to the kernels that they name."""
import numpy as np
import pytest

import f8_plain as p
from f8_plain import HALF24
from test_gpu_f8 import gate_up, largest_cut, product, put
from test_gpu_f8_gated import matrix as of_scale
from test_gpu_f8_gated import small

pytestmark = pytest.mark.gpu

TILES = [  # type, tokens, cols, rows; a tile's tokens and rows, the most tiles of a workgroup, steps
    ("f32", 1100, 100, 7003, 128, 128, 1, 1), ("f32", 1310, 250, 10985, 128, 128, 2, 2), ("f32", 2066, 380, 7180, 128, 128, 2, 3),
    ("f32", 8707, 380, 1821, 128, 128, 3, 3), ("f32", 1330, 2040, 10877, 256, 128, 2, 16), ("f32", 1284, 1900, 10761, 256, 128, 2, 15),
    ("f32", 2062, 2800, 9617, 256, 128, 3, 22), ("f32", 2050, 100, 5003, 256, 256, 1, 1), ("f32", 3210, 250, 7607, 256, 256, 2, 2),
    ("f32", 1804, 380, 10959, 256, 256, 2, 3), ("f32", 3225, 380, 9985, 256, 256, 3, 3),
    ("bf16", 1000, 100, 2005, 64, 64, 1, 1), ("bf16", 903, 250, 8397, 64, 64, 2, 2), ("bf16", 650, 380, 10907, 64, 64, 2, 3),
    ("bf16", 7285, 250, 2183, 64, 64, 4, 2), ("bf16", 540, 100, 11137, 128, 128, 1, 1), ("bf16", 1299, 250, 10901, 128, 128, 2, 2),
    ("bf16", 1293, 380, 11058, 128, 128, 2, 3), ("bf16", 4354, 380, 7258, 128, 128, 4, 3), ("bf16", 385, 100, 9426, 256, 128, 1, 1),
    ("bf16", 1861, 250, 8710, 256, 128, 3, 2), ("bf16", 1413, 380, 10948, 256, 128, 3, 3), ("bf16", 780, 100, 10127, 256, 256, 1, 1),
    ("bf16", 3622, 250, 10898, 256, 256, 3, 2), ("bf16", 2068, 380, 11058, 256, 256, 2, 3)]
GATED = [
    ("gated", 1500, 100, 2003, 128, 128, 1, 1), ("gated", 533, 250, 11169, 128, 128, 2, 2), ("gated", 1042, 250, 7170, 128, 128, 3, 2),
    ("gated", 662, 380, 10968, 128, 128, 3, 3), ("gated", 2000, 100, 3003, 256, 128, 1, 1), ("gated", 1167, 250, 9938, 256, 128, 2, 2),
    ("gated", 2574, 250, 7782, 256, 128, 3, 2), ("gated", 8843, 380, 1287, 256, 128, 2, 3), ("gated", 4496, 380, 4481, 256, 128, 3, 3),
    ("gated", 4000, 1100, 3990, 256, 128, 2, 9)]


def case(v):
    return "-".join(str(x) for x in v[:6]) if isinstance(v, tuple) else None


def up(n, m):
    return -(-n // m) * m


def exact(X, W):
    """Every partial sum is exact in f32."""
    return X[2].astype(np.float32) @ W[2].astype(np.float32).T


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("c", TILES, ids=case)
def test_tiles(backend, c, aligned):
    """Aligned outputs leave 16 bytes a lane, others one by one."""
    type, tokens, cols, rows = c[:4]
    rng = np.random.default_rng(tokens + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    stride, offset = (up(rows, 8) + 8, 8) if aligned else (rows + rows % 2 + 1, 3)
    got, rest = product(backend, X, W, tokens, cols, rows, type, stride, offset)
    want = exact(X, W)
    assert np.array_equal(got, want if type == "f32" else p.bf16(want).astype(np.float32))
    assert np.all(rest == -7)


@pytest.mark.parametrize("where", ["apart", "Y"])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("c", [c for c in TILES if c[0] == "f32"], ids=case)
def test_tiles_residual(backend, c, aligned, where):
    """R in a buffer of its own, and in Y: each of its values once, at its output's place."""
    type, tokens, cols, rows = c[:4]
    rng = np.random.default_rng(tokens + cols)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    stride, offset = (up(rows, 4) + 4, 4) if aligned else (rows + rows % 2 + 1, 3)
    r = rng.integers(-2 ** 15, 2 ** 15, tokens * stride + offset + 3).astype(np.float32) / 8
    R = put(backend, r)
    got, rest = product(backend, X, W, tokens, cols, rows, "f32", stride, offset, residual=R, Y=R if where == "Y" else None)
    slots = offset + np.arange(tokens)[:, None] * stride + np.arange(rows)
    assert np.array_equal(got, r[slots] + exact(X, W))
    left = np.ones(len(r), bool)
    left[slots] = False
    assert np.array_equal(rest, r[left] if where == "Y" else np.full(left.sum(), -7, np.float32))


@pytest.mark.parametrize("c", [c for c in TILES if c[6] > 1 and c[7] <= 3], ids=case)
def test_tiles_special(backend, c):
    """NaN codes of a token and of a row, within the first tile and at the last one's end, poison their own outputs alone;
    scales at both ends of the range, and sums past f32's."""
    type, tokens, cols, rows = c[:4]
    rng = np.random.default_rng(rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    W[1][:, 0], W[1][:, 1: p.blocks(cols, 128)] = 237, 0  # 2^110 and 2^-127
    X[1][2, 0], X[1][0, 0] = 17, 245                      # 2^-110 and 2^118
    X[0][1, 7] = X[0][tokens - 1, cols - 1] = 0x7f
    W[0][33, cols - 10] = W[0][rows - 1, 0] = 0xff
    got, rest = product(backend, X, W, tokens, cols, rows, type, up(rows, 8), 0)
    tokens_ok, rows_ok = np.setdiff1d(np.arange(tokens), [1, tokens - 1]), np.setdiff1d(np.arange(rows), [33, rows - 1])
    nan = np.isnan(got)
    assert nan[[1, tokens - 1]].all() and nan[:, [33, rows - 1]].all()
    # the first block alone counts, whole numbers times a power of two; what the others add is below 2^-110
    a, b = (np.where(np.isnan(v), 0, v).astype(np.float32) for v in (p.CODES[X[0][:, :128]], p.CODES[W[0][:, :128]]))
    first = (a @ b.T)[tokens_ok][:, rows_ok]
    g = got[tokens_ok][:, rows_ok]
    assert not np.isfinite(g[0])[first[0] != 0].any()
    first, g = first[1:], g[1:]
    scale = 2.0 ** (X[1][tokens_ok[1:], :1].astype(np.float64) - 127 + 110)
    want = (first * scale).astype(np.float32)
    want = want if type == "f32" else p.bf16(want).astype(np.float32)
    assert np.array_equal(g[first != 0], want[first != 0])
    assert np.all(np.abs(g[first == 0]) < 2.0 ** -100)
    assert np.all(rest == -7)


@pytest.mark.parametrize("c", GATED, ids=case)
def test_gated_tiles(backend, c):
    tokens, cols, ff = c[1:4]
    rng = np.random.default_rng(tokens + ff)
    X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    Wg[1][:] -= 5
    p.check_f8(*gate_up(backend, X, Wg, Wu, tokens, cols, ff), p.silu(exact(X, Wg).astype(np.float64) / 32) * exact(X, Wu), 8 * HALF24)


@pytest.mark.parametrize("c", [c for c in GATED if c[6] > 1], ids=case)
def test_gated_tiles_special(backend, c):
    """NaN codes in the first tile and at the last one's end: their outputs alone, and no scale sees them."""
    tokens, cols, ff = c[1:4]
    rng = np.random.default_rng(ff)
    X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    Wg[1][:] -= 5
    want = p.silu(exact(X, Wg).astype(np.float64) / 32) * exact(X, Wu)
    X[0][1, 7] = X[0][tokens - 1, cols - 1] = 0x7f
    Wg[0][33, cols - 10], Wu[0][ff - 1, 0] = 0xff, 0x7f
    codes, scales = gate_up(backend, X, Wg, Wu, tokens, cols, ff)
    bad = np.zeros((tokens, ff), bool)
    bad[[1, tokens - 1]] = bad[:, [33, ff - 1]] = True
    assert np.array_equal(np.isnan(p.CODES[codes[:, :ff]]), bad)
    assert np.all(scales[[1, tokens - 1]] == 127)
    want[bad] = 0
    codes = codes.copy()
    codes[:, :ff][bad] = 0
    p.check_f8(codes, scales, want, 8 * HALF24)


@pytest.mark.parametrize("type,tokens,cols,rows", [("f32", 2066, 380, 7180), ("bf16", 1293, 380, 11058), ("f32", 205, 2600, 2503)])
def test_same_call_same_bits(backend, type, tokens, cols, rows):
    """The same call gives the same bits. (Another number of tokens may take another kernel and another order of sums.)"""
    rng = np.random.default_rng(9)
    X, W = p.ordinary(rng, tokens, cols, 1), p.ordinary(rng, rows, cols, 128)
    first, _ = product(backend, X, W, tokens, cols, rows, type, rows, 0)
    for _ in range(2):
        again, _ = product(backend, X, W, tokens, cols, rows, type, rows, 0)
        assert np.array_equal(first, again)


@pytest.mark.parametrize("tokens,cols,rows", [(5, 260, 200), (205, 1000, 2503), (903, 250, 8397), (1413, 380, 10948), (2068, 380, 11058)])
def test_cancelling_products(backend, tokens, cols, rows):
    """Two products of up to 2^17 that cancel in every eight, and whole numbers below 64 beside them: exact to f32; to
    bf16, off by what is cut from the products, 7 * 2^-13 of their magnitudes, and one rounding."""
    rng = np.random.default_rng(tokens)
    x, w = small(rng, tokens, cols), small(rng, rows, cols)
    x[:, 0:cols - 8:8], x[:, 1:cols - 8:8] = 256, -256
    w[:, 1:cols - 8:8] = w[:, 0:cols - 8:8] = rng.choice([-448, 256, 448], (rows, len(range(0, cols - 8, 8))))
    X, W = of_scale(x, 1, 127), of_scale(w, 128, 127)
    want = exact(X, W).astype(np.float64)
    got, _ = product(backend, X, W, tokens, cols, rows, "f32", rows, 0)
    assert np.array_equal(got, want)
    got, _ = product(backend, X, W, tokens, cols, rows, "bf16", rows, 0)
    sums = (128 + p.blocks(cols, 128) + 8) * 2.0 ** -23 * (np.abs(X[2]) @ np.abs(W[2]).T)
    assert np.all(np.abs(got - want) <= (sums + largest_cut(X[2], W[2])) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want))
