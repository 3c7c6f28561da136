"""The 8-bit floating-point operators on the GPU at the largest sizes: dimensions of 2^21, buffers and outputs whose
offsets pass 32 bits, and a captured call of persistent tiles. What lies far out is written and read on its own."""
import numpy as np
import pytest

import f8_plain as p
from f8_plain import HALF24
from test_gpu_f8 import F8, get, product, put

pytestmark = pytest.mark.gpu

MAX = 2 ** 21


@pytest.fixture
def be(backend):
    """The context; what a test allocates is freed with it."""
    before = set(backend.buffers)
    yield backend
    for b in set(backend.buffers) - before:
        backend.free(b)


def zeros(be, nbytes):
    return be.alloc_bytes(nbytes, zero=True)


def part(be, buf, dtype, at, n):
    size = np.dtype(dtype).itemsize
    return be.read_bytes(buf, n * size, at * size).view(dtype)


def ends(rows):
    """The first and the last 256 rows of many (2^21 of them are whole blocks of 128)."""
    return [slice(0, rows)] if rows < 512 else [slice(0, 256), slice(rows - 256, rows)]


# ----------------------------------------------------- dimensions of 2^21
@pytest.mark.parametrize("rows,cols,block", [(1, MAX, 1), (3, MAX, 128), (MAX, 1, 1), (MAX, 1, 128)])
def test_quantize_long(be, rows, cols, block):
    x = np.random.default_rng(rows).normal(0, 1, (rows, cols)).astype(np.float32)
    out = F8(be, rows, cols, block)
    be.f8_quantize(put(be, x), rows, cols, block, out.codes, out.scales)
    codes, scales = out.read()
    for at in ends(rows):
        want, want_scales = p.quantize(x[at].astype(np.float64), block)
        assert np.array_equal(p.CODES[codes[at]], want)
        assert np.array_equal(scales[at.start // block: -(-at.stop // block)], want_scales)


@pytest.mark.parametrize("rows,cols", [(2, MAX), (2, MAX - 3), (MAX, 1), (MAX, 4)])
def test_norm_long(be, rows, cols):
    rng = np.random.default_rng(cols)
    x, r = (rng.normal(0, 1, (rows, cols)).astype(np.float32) for _ in range(2))
    gamma = rng.normal(1, 0.2, cols).astype(np.float32)
    out, R = F8(be, rows, cols), put(be, r)
    be.f8_norm(put(be, x), put(be, gamma), 1e-6, rows, cols, out.codes, out.scales, residual=R, H=R)
    h = x + r
    assert np.array_equal(get(be, R, np.float32, (rows, cols)), h)
    codes, scales = out.read()
    for at in ends(rows):
        v = h[at].astype(np.float64)
        y = v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * gamma.astype(np.float64)
        p.check_f8(codes[at], scales[at], y, 4 * HALF24)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,cols,rows", [(3, MAX, 17), (40, MAX - 100, 33), (1, 1, MAX), (MAX, 5, 3)])
def test_project_long(be, tokens, cols, rows, type):
    rng = np.random.default_rng(tokens + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    got, rest = product(be, X, W, tokens, cols, rows, type, rows + 1, 1)
    want = X[2] @ W[2].T
    assert np.abs(want).max() < 2 ** 17  # in steps of 2^-6: exact in f32
    assert np.array_equal(got, want.astype(np.float32) if type == "f32" else p.bf16(want).astype(np.float32))
    assert np.all(rest == -7)


# ------------------------------------------------- offsets past 32 bits
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_far(be, block):
    """2^20 and some rows of 4100 bf16 values: 8.6 GB to 4.4 GB."""
    rows, cols = 2 ** 20 + 7, 4100
    pitch, spitch, up = p.layout(rows, cols, block)
    last = np.random.default_rng(1).normal(0, 1, (7, cols))
    X, codes, scales = zeros(be, rows * cols * 2), zeros(be, rows * pitch), zeros(be, up * spitch)
    be.write_bytes(X, p.bf16_bits(last).reshape(-1).view(np.uint8), (rows - 7) * cols * 2)
    be.f8_quantize(X, rows, cols, block, codes, scales, type="bf16")
    want, want_scales = p.quantize(p.bf16(last), block)  # 2^20 is a multiple of 128: the last rows' block holds them alone
    got = part(be, codes, np.uint8, (rows - 7) * pitch, 7 * pitch).reshape(7, pitch)
    assert np.array_equal(p.CODES[got], want)
    n = len(want_scales)
    assert np.array_equal(part(be, scales, np.uint8, (up - n) * spitch, n * spitch).reshape(n, spitch), want_scales)


def test_norm_far(be):
    """The same of the norm with H in place of R: 8.6 GB each of X and H."""
    rows, cols = 2 ** 19 + 3, 4100
    pitch, spitch, _ = p.layout(rows, cols, 1)
    rng = np.random.default_rng(2)
    x, r = (rng.normal(0, 1, (3, cols)).astype(np.float32) for _ in range(2))
    X, R, codes, scales = zeros(be, rows * cols * 4), zeros(be, rows * cols * 4), zeros(be, rows * pitch), zeros(be, rows * spitch)
    for buf, v in ((X, x), (R, r)):
        be.write_bytes(buf, v.reshape(-1).view(np.uint8), (rows - 3) * cols * 4)
    be.f8_norm(X, put(be, np.ones(cols, np.float32)), 1e-6, rows, cols, codes, scales, residual=R, H=R)
    h = x + r
    assert np.array_equal(part(be, R, np.float32, (rows - 3) * cols, 3 * cols).reshape(3, cols), h)
    h = h.astype(np.float64)
    p.check_f8(part(be, codes, np.uint8, (rows - 3) * pitch, 3 * pitch).reshape(3, pitch),
               part(be, scales, np.uint8, (rows - 3) * spitch, 3 * spitch).reshape(3, spitch),
               h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6), 4 * HALF24)


def far_matrix(be, rows, cols, block, some):
    """Buffers of a matrix of zeros whose last rows are `some`: their codes, and scales of 1 (or, of 128 rows, their own)."""
    pitch, spitch, up = p.layout(rows, cols, block)
    n = len(some[0])
    codes, scales = zeros(be, rows * pitch), put(be, np.full(up * spitch, 127, np.uint8))
    be.write_bytes(codes, some[0].reshape(-1), (rows - n) * pitch)
    return codes, scales


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_project_far_weights(be, tokens, type):
    """Weights of 4.6 GB, 2^21 rows of 2100 columns; the last 200 are not zero."""
    cols, rows, n = 2100, MAX, 200
    rng = np.random.default_rng(tokens)
    X, some = p.matrix(rng, tokens, cols, 1), p.matrix(rng, n, cols, 128)
    some = (some[0], None, p.values(some[0], np.full_like(some[1], 127), 128)[:, :cols])
    W, Ws = far_matrix(be, rows, cols, 128, some)
    size = 4 if type == "f32" else 2
    Y = be.alloc_bytes(tokens * rows * size)
    be.f8_project(put(be, X[0]), put(be, X[1]), tokens, cols, W, Ws, rows, Y, type=type)
    want = X[2] @ some[2].T
    for t in {0, tokens // 2, tokens - 1}:
        row = part(be, Y, np.float32 if type == "f32" else np.uint16, t * rows, rows)
        row = row if type == "f32" else p.from_bf16(row)
        assert np.all(row[: rows - n] == 0)
        assert np.array_equal(row[rows - n:], (want[t] if type == "f32" else p.bf16(want[t])).astype(np.float32))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,rows", [(3, 200), (520, 9000)])
def test_project_far_outputs(be, tokens, rows, type):
    """A stride that puts the last tokens' outputs past 2^32 values."""
    cols = 260
    stride, offset = (2 ** 32 // (tokens - 1)) + 8 & ~7, 8
    rng = np.random.default_rng(rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    dtype = np.float32 if type == "f32" else np.uint16
    Y = be.alloc_bytes(((tokens - 1) * stride + offset + rows + 8) * np.dtype(dtype).itemsize)
    mark = np.full(rows + 16, 7, dtype)
    at = [t * stride + offset for t in (0, tokens // 2, tokens - 1)]
    for a in at:
        be.write_bytes(Y, mark.view(np.uint8), (a - 8) * mark.itemsize)
    be.f8_project(put(be, X[0]), put(be, X[1]), tokens, cols, put(be, W[0]), put(be, W[1]), rows, Y, type=type, stride=stride,
                  offset=offset)
    assert (tokens - 1) * stride >= 2 ** 32
    for a, t in zip(at, (0, tokens // 2, tokens - 1)):
        got = part(be, Y, dtype, a - 8, rows + 16)
        assert np.array_equal(got[:8], mark[:8]) and np.array_equal(got[-8:], mark[:8])
        want = X[2][t] @ W[2].T
        got = got[8:-8] if type == "f32" else p.from_bf16(got[8:-8])
        assert np.array_equal(got, (want if type == "f32" else p.bf16(want)).astype(np.float32))


@pytest.mark.parametrize("tokens", [1, 300])
def test_gate_up_far(be, tokens):
    """Two matrices of 4.6 GB."""
    cols, ff, n = 2100, MAX, 256
    rng = np.random.default_rng(tokens)
    X, g, u = p.matrix(rng, tokens, cols, 1), p.matrix(rng, n, cols, 128), p.matrix(rng, n, cols, 128)
    g, u = ((m[0], None, p.values(m[0], np.full_like(m[1], 127), 128)[:, :cols]) for m in (g, u))
    (Wg, Wgs), (Wu, Wus) = far_matrix(be, ff, cols, 128, g), far_matrix(be, ff, cols, 128, u)
    pitch, spitch, _ = p.layout(tokens, ff, 1)
    codes, scales = be.alloc_bytes(tokens * pitch), be.alloc_bytes(tokens * spitch)
    ws = be.alloc_bytes(be.f8_gate_up_workspace_bytes(tokens, ff))
    be.f8_gate_up(put(be, X[0]), put(be, X[1]), tokens, cols, Wg, Wgs, Wu, Wus, ff, codes, scales, ws)
    want = p.silu(X[2] @ g[2].T) * (X[2] @ u[2].T)
    for t in {0, tokens // 2, tokens - 1}:
        c, s = part(be, codes, np.uint8, t * pitch, pitch), part(be, scales, np.uint8, t * spitch, spitch)
        assert np.all(c[: ff - n] & 127 == 0) and np.all(s[: (ff - n) // 128] == 127)
        p.check_f8(c[None, ff - n:], np.concatenate([s[(ff - n) // 128:], [127, 127]])[None], want[t:t + 1], 8 * HALF24)


# --------------------------------------------------------- a captured call
def test_captured_tiles(be):
    """A gated pair and a projection in persistent tiles, replayed with other inputs and eager calls between."""
    tokens, width, ff = 1167, 250, 9938
    rng = np.random.default_rng(7)
    Wg, Wu, Wd = p.matrix(rng, ff, width, 128), p.matrix(rng, ff, width, 128), p.matrix(rng, width, ff, 128)
    Wg[1][:] -= 5
    Xs = [p.matrix(rng, tokens, width, 1) for _ in range(3)]
    X = [put(be, a) for a in Xs[0][:2]]
    w = [put(be, a) for m in (Wg, Wu, Wd) for a in m[:2]]
    out, ws = F8(be, tokens, ff), be.alloc_bytes(be.f8_gate_up_workspace_bytes(tokens, ff))
    Y = put(be, np.zeros((tokens, width), np.float32))

    def run():
        be.f8_gate_up(X[0], X[1], tokens, width, w[0], w[1], w[2], w[3], ff, out.codes, out.scales, ws)
        be.f8_project(out.codes, out.scales, tokens, ff, w[4], w[5], width, Y)

    run()
    be.idle()
    be.graph_begin()
    run()
    graph = be.graph_end()
    for k in (0, 1, 2, 1, 0):
        for buf, a in zip(X, Xs[k][:2]):
            be.write_bytes(buf, a.reshape(-1))
        be.graph_launch(graph)
        replayed, codes = get(be, Y, np.float32, (tokens, width)), out.read()
        g, u = Xs[k][2] @ Wg[2].T / 32, Xs[k][2] @ Wu[2].T
        p.check_f8(*codes, p.silu(g) * u, 8 * HALF24)
        run()
        assert np.array_equal(get(be, Y, np.float32, (tokens, width)), replayed)
        assert all(np.array_equal(a, b) for a, b in zip(out.read(), codes))
    be.graph_free(graph)
