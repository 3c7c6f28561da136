"""The gated pair on the GPU where f32 sums matter, against 64 bits (f8_plain): inputs whose sums are exact in f32 in any
order, in calls of every number of tokens."""
import numpy as np
import pytest

import f8_plain as p
from f8_plain import HALF24
from test_gpu_f8 import gate_up

pytestmark = pytest.mark.gpu

# 16 x 16 and 32 x 16 outputs of shared columns, and tiles of 128 and of 256 tokens
SIZES = [(3, 300, 200), (131, 260, 1003), (1990, 384, 2000), (4000, 900, 3990)]


def small(rng, rows, cols):
    """Code values [rows, pitch] of 0, +-1 and +-2, 0 past `cols`."""
    v = np.zeros((rows, 128 * p.blocks(cols, 128)))
    v[:, :cols] = rng.integers(-2, 3, (rows, cols))
    return v


def matrix(v, block, byte):
    """(code bytes, scale bytes, values) with one scale."""
    rows, pitch = v.shape
    _, spitch, up = p.layout(rows, pitch, block)
    scales = np.full((up, spitch), 127, np.uint8)
    scales[:, : pitch // 128] = byte
    return p.of_values(v, scales, block, pitch)


@pytest.mark.parametrize("tokens,cols,ff", SIZES)
def test_gate_up_cancelled(backend, tokens, cols, ff):
    """Two products of 2^17 that cancel in every eighth neighbours, beside sums of at most some hundred: what is left is
    exact, and finite."""
    rng = np.random.default_rng(tokens)
    x, g, u = small(rng, tokens, cols), small(rng, ff, cols), small(rng, ff, cols)
    x[:, 0:cols - 8:8], x[:, 1:cols - 8:8] = 256, -256
    for w in (g, u):
        w[:, 1:cols - 8:8] = w[:, 0:cols - 8:8] = rng.choice([-448, 256, 448], (ff, len(range(0, cols - 8, 8))))
    X, Wg, Wu = matrix(x, 1, 127), matrix(g, 128, 122), matrix(u, 128, 127)  # gates of about 1
    codes, scales = gate_up(backend, X, Wg, Wu, tokens, cols, ff)
    assert not np.isnan(p.CODES[codes]).any()
    # every product and sum is a whole number below 2^24 (of 2^-5 in the gates): at most 2 * 448 * 256 and the rest
    a = x.astype(np.float32) @ g.astype(np.float32).T
    b = x.astype(np.float32) @ u.astype(np.float32).T
    p.check_f8(codes, scales, p.silu(a.astype(np.float64) / 32) * b, 8 * HALF24)


@pytest.mark.parametrize("tokens,cols,ff", SIZES)
def test_gate_up_scale_of_many_near_its_border(backend, tokens, cols, ff):
    """All columns of a block within 2^-13 of a scale's border, one of them, not among its first, past it."""
    x, g, u = (np.zeros((n, 128 * p.blocks(cols, 128))) for n in (tokens, ff, ff))
    rng = np.random.default_rng(ff)
    past = np.arange(ff) % 128 == 100
    x[:, 0], x[:, 9], x[:, 200] = 256, 1, 1
    u[:, 0], u[:, 9] = 56, np.where(past, 1, -1)  # 1.75 * 2^13, and one more or one less
    g[:, 200] = 32  # silu(32) = 32 in f32
    x[:, 64:128] = rng.integers(0, 3, (tokens, 64))  # meets zeros
    X, Wg, Wu = matrix(x, 1, 127), matrix(g, 128, 127), matrix(u, 128, 127)
    codes, scales = gate_up(backend, X, Wg, Wu, tokens, cols, ff)
    h = np.broadcast_to(32.0 * (14336 + np.where(past, 1, -1)), (tokens, ff))
    p.check_f8(codes, scales, h, 8 * HALF24)
    holds = np.bincount(np.arange(ff) // 128, past) > 0
    assert np.array_equal(scales[:, : len(holds)], np.broadcast_to(np.where(holds, 138, 137), (tokens, len(holds))))


@pytest.mark.parametrize("tokens", [3, 131, 1000, 3000])
def test_gate_up_far_gates(backend, tokens):
    """One product a sum: gates from -88 to -192, whose exp passes f32's range, with up to 2^121 of u so that the products
    lie inside it and decide their blocks' scales."""
    cols, ff = 128, 7 * 128
    gates = {0: (-88, -96), 20: (-88, -96, -104), 60: (-96, -104, -112, -120), 100: (-104, -112, -128, -144),
             110: (-112, -128, -144, -160), 120: (-128, -144, -160, -176), 121: (-176, -192)}
    rng = np.random.default_rng(tokens)
    x, g, u = np.zeros((tokens, cols)), np.zeros((ff, cols)), np.zeros((ff, cols))
    at = np.arange(tokens) % cols
    x[np.arange(tokens), at] = 1
    X = matrix(x, 1, 127)
    u[:] = rng.choice([1, 1.25, -1.75], (ff, cols))
    scales = np.full((ff // 128, 4), 127, np.uint8)
    for b, (k, choice) in enumerate(gates.items()):
        g[b * 128:(b + 1) * 128] = rng.choice(choice, (128, cols))
        scales[b, 0] = 127 + k
    Wg, Wu = matrix(g, 128, 127), p.of_values(u, scales, 128, cols)
    codes, got = gate_up(backend, X, Wg, Wu, tokens, cols, ff)
    a, b = g[:, at].T, Wu[2][:, at].T
    h = a / (1 + np.exp(-a)) * b
    assert np.abs(h).reshape(tokens, -1, 128).max((0, 2)).min() > 2.0 ** -133  # every block has values that f32 holds
    p.check_f8(codes, got, h, 8 * HALF24)
