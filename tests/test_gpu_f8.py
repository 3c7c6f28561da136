"""The 8-bit floating-point operators on the GPU against their definitions in 64
bits (f8_plain): conversion, norm with the residual, projection, gated pair, and a
feed-forward block made of them."""
import numpy as np
import pytest

import f8_plain as p
from f8_plain import HALF24

pytestmark = pytest.mark.gpu


def put(be, a):
    a = np.ascontiguousarray(a)
    buf = be.alloc_bytes(a.nbytes)
    be.write_bytes(buf, a.reshape(-1).view(np.uint8))
    return buf


def get(be, buf, dtype, shape):
    n = int(np.prod(shape)) * np.dtype(dtype).itemsize
    return be.read_bytes(buf, n).view(dtype).reshape(shape)


class F8:
    """An f8 matrix's buffers, filled with 0xAA and two bytes longer than it needs."""

    def __init__(self, be, rows, cols, block=1):
        self.be, self.shape = be, p.layout(rows, cols, block)
        self.rows = rows
        codes, scales = be.f8_bytes(rows, cols, block)
        assert (codes, scales) == (rows * self.shape[0], self.shape[2] * self.shape[1])
        self.codes = put(be, np.full(codes + 2, 0xAA, np.uint8))
        self.scales = put(be, np.full(scales + 2, 0xAA, np.uint8))

    def read(self):
        pitch, spitch, up = self.shape
        c, s = self.be.read_bytes(self.codes), self.be.read_bytes(self.scales)
        assert np.all(c[-2:] == 0xAA) and np.all(s[-2:] == 0xAA)
        return c[:-2].reshape(self.rows, pitch), s[:-2].reshape(up, spitch)


def as_type(x, type):
    """x in the type, as (array to upload, its values in f64)"""
    if type == "bf16":
        return p.bf16_bits(x), p.bf16(x)
    x = x.astype(np.float32)
    return x, x.astype(np.float64)


def hidden(rng, rows, cols):
    x = rng.normal(0, 1, (rows, cols)) * np.exp(rng.normal(0, 0.8, cols))
    return np.where(rng.random((rows, cols)) < 0.001, 8 * x, x)


# ------------------------------------------------------------------ quantize
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 6144), (3, 127), (2, 128), (5, 129), (127, 500), (128, 512), (129, 260),
                                       (300, 1030), (7, 2564)])
def test_quantize(backend, rows, cols, block, type):
    rng = np.random.default_rng(rows * 7 + cols)
    data, x = as_type(hidden(rng, rows, cols) * 10.0 ** rng.integers(-6, 6, (rows, 1)), type)
    out = F8(backend, rows, cols, block)
    backend.f8_quantize(put(backend, data), rows, cols, block, out.codes, out.scales, type=type)
    codes, scales = out.read()
    want, want_scales = p.quantize(x, block)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(p.CODES[codes], want)


@pytest.mark.parametrize("block", [1, 128])
def test_quantize_edges(backend, block):
    """Every power of two and the scale's border beside it, subnormals, zeros of both signs, rows of zeros, and
    values that are not finite: NaN, with the scale of the others."""
    cols = 128
    rows = []
    for e in range(-149, 128):
        top = np.float32(2.0 ** e)
        for amax in (top, np.float32(min(1.75 * 2.0 ** e, 3.4e38)), np.nextafter(np.float32(1.75 * 2.0 ** e), np.float32(3e38)),
                     np.nextafter(top, np.float32(0))):
            r = np.linspace(-1, 1, cols).astype(np.float32) * amax
            r[5] = amax
            rows.append(r)
    rows.append(np.zeros(cols, np.float32))
    rows.append(np.full(cols, -0.0, np.float32))
    for special in (np.inf, -np.inf, np.nan):
        r = np.linspace(-3, 5, cols).astype(np.float32)
        r[[0, 77]] = special
        rows.append(r)
        rows.append(np.full(cols, special, np.float32))
    x = np.stack(rows)
    out = F8(backend, len(x), cols, block)
    backend.f8_quantize(put(backend, x), len(x), cols, block, out.codes, out.scales)
    codes, scales = out.read()
    want, want_scales = p.quantize(x.astype(np.float64), block)
    assert np.array_equal(scales, want_scales)
    got = p.CODES[codes]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
    assert np.array_equal(np.signbit(got[~np.isnan(want)]), np.signbit(want[~np.isnan(want)]))


# ---------------------------------------------------------------------- norm
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2560), (4, 100), (3, 129), (5, 255), (9, 512), (2, 1030), (33, 2560),
                                       (3, 4099), (2, 8192), (2, 16384), (2, 20000), (1, 33333)])
@pytest.mark.parametrize("residual,H", [("none", "none"), ("none", "new"), ("own", "new"), ("own", "R"), ("own", "none"),
                                        ("own", "X"), ("none", "X")])
def test_norm(backend, rows, cols, type, residual, H):
    if H == "X" and type == "bf16":
        pytest.skip("H may be X only where X is f32")
    rng = np.random.default_rng(rows * 31 + cols)
    data, x = as_type(hidden(rng, rows, cols), type)
    r = hidden(rng, rows, cols).astype(np.float32)
    gamma = rng.normal(1, 0.2, cols).astype(np.float32)
    X, R, out = put(backend, data), put(backend, r), F8(backend, rows, cols)
    new = put(backend, np.full(rows * cols + 1, -7, np.float32))
    Hbuf = {"none": None, "new": new, "R": R, "X": X}[H]
    backend.f8_norm(X, put(backend, gamma), 1e-6, rows, cols, out.codes, out.scales,
                    residual=R if residual == "own" else None, H=Hbuf, type=type)
    h = x.astype(np.float32) + r if residual == "own" else x.astype(np.float32)
    if Hbuf is not None:
        assert np.array_equal(get(backend, Hbuf, np.float32, (rows, cols)).view(np.uint32), h.view(np.uint32))
    assert get(backend, new, np.float32, (rows * cols + 1,))[-1] == -7
    h = h.astype(np.float64)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6) * gamma.astype(np.float64)
    # 1/sqrt rounded to f32, times h, times gamma: three roundings; eps is f32(1e-6) there, 2^-25 of it off
    p.check_f8(*out.read(), y, 4 * HALF24)


def test_norm_values(backend):
    """Rows of zeros, of large values (their squares pass f32), of tiny ones (eps decides), with infinities and NaN;
    eps 0 on a row of zeros gives NaN, as the formula does."""
    cols = 300
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (7, cols)).astype(np.float32)
    x[1] = 0
    x[2] *= np.float32(1e25)
    x[3] *= np.float32(1e-30)
    x[4, 17] = np.inf
    x[5, 250] = np.nan
    gamma = np.ones(cols, np.float32)
    X, g = put(backend, x), put(backend, gamma)
    out = F8(backend, 7, cols)
    backend.f8_norm(X, g, 1e-6, 7, cols, out.codes, out.scales)
    codes, scales = out.read()
    h = x.astype(np.float64)
    fine = [0, 1, 2, 3, 6]
    with np.errstate(invalid="ignore"):
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6)
    p.check_f8(codes[fine], scales[fine], y[fine], 4 * HALF24)
    got = p.CODES[codes]
    assert np.isnan(got[4, 17]) and np.all(np.delete(got[4], 17) == 0)
    assert np.all(np.isnan(got[5, :cols])) and np.all(got[5, cols:] == 0)
    backend.f8_norm(X, g, 0.0, 7, cols, out.codes, out.scales)
    assert np.all(np.isnan(p.CODES[out.read()[0]][1, :cols]))


# ------------------------------------------------------------------- project
SHAPES = [  # tokens, cols, rows
    (1, 1, 1), (1, 128, 16), (1, 2560, 300), (1, 129, 17), (2, 500, 127), (15, 1030, 128), (16, 256, 129), (17, 384, 515),
    (33, 640, 64), (63, 2560, 100), (64, 130, 33), (65, 260, 257), (100, 1152, 300), (127, 128, 130), (128, 512, 128),
    (129, 1024, 384), (200, 700, 1000), (256, 256, 256), (257, 300, 513), (300, 2560, 640), (511, 128, 2000), (513, 1500, 385),
    (1025, 256, 1030), (1500, 384, 2050), (2100, 130, 4100)]


def product(backend, X, W, tokens, cols, rows, type, stride, offset, residual=None, Y=None):
    n = tokens * stride + offset + 3
    if Y is None:
        fill = np.full(n, -7, np.float32)
        Y = put(backend, fill if type == "f32" else p.bf16_bits(fill))
    backend.f8_project(put(backend, X[0]), put(backend, X[1]), tokens, cols, put(backend, W[0]), put(backend, W[1]), rows, Y,
                       residual=residual, type=type, stride=stride, offset=offset)
    flat = get(backend, Y, np.float32, (n,)) if type == "f32" else p.from_bf16(get(backend, Y, np.uint16, (n,)))
    slots = offset + np.arange(tokens)[:, None] * stride + np.arange(rows)
    rest = np.ones(n, bool)
    rest[slots] = False
    return flat[slots], flat[rest]


@pytest.mark.parametrize("tokens,cols,rows", SHAPES)
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("extra,offset", [(0, 0), (3, 2), (4, 4)])
def test_project_exact(backend, tokens, cols, rows, type, extra, offset):
    """Values whose sums are exact in any order: every product counts once, and nothing else is written."""
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    got, rest = product(backend, X, W, tokens, cols, rows, type, rows + extra, offset)
    want = X[2] @ W[2].T
    assert np.array_equal(got, want.astype(np.float32) if type == "f32" else p.bf16(want).astype(np.float32))
    assert np.all(rest == -7)


@pytest.mark.parametrize("tokens,cols,rows", SHAPES)
def test_project_residual(backend, tokens, cols, rows):
    """R in a buffer of its own and in Y itself."""
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    stride, offset = rows + 1, 1
    r = rng.normal(0, 100, tokens * stride + offset + 3).astype(np.float32)
    slots = offset + np.arange(tokens)[:, None] * stride + np.arange(rows)
    sums = (X[2] @ W[2].T).astype(np.float32)
    R = put(backend, r)
    for Y in (None, R):
        got, rest = product(backend, X, W, tokens, cols, rows, "f32", stride, offset, residual=R, Y=Y)
        assert np.array_equal(got, r[slots] + sums)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,cols,rows", [
    (2000, 300, 2500),   # tiles of 256 x 128 (f32: 128 x 128) in one round
    (2100, 300, 10300),  # of 256 x 128 in three, three steps a tile: the next tile begins in the other buffer (f32: 256 x 256 in two)
    (2100, 3840, 9600),  # 128 x 128 tiles, two a CU, in two and a half rounds (f32 too)
    (1000, 260, 10200),  # 256 x 256 tiles in one round (f32 too, and in the next three)
    (5600, 300, 5800),   # and in two, three steps a tile
    (5600, 200, 5800),   # two steps
    (5600, 100, 5800),   # one step: a tile a workgroup
    (700, 513, 2100),    # 64 x 64 tiles, two to four a CU (f32: shared columns, 32 x 64)
    (1100, 640, 4200)])  # 256 x 128 (f32: 128 x 128)
def test_project_exact_many(backend, tokens, cols, rows, type):
    """The same over sizes that every tile takes, over several rounds; rows and tokens past the last tile's middle."""
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    got, rest = product(backend, X, W, tokens, cols, rows, type, rows + 8, 8)
    want = (X[2].astype(np.float32) @ W[2].astype(np.float32).T)  # exact in f32: every partial sum is
    assert np.array_equal(got, want if type == "f32" else p.bf16(want).astype(np.float32))
    assert np.all(rest == -7)


def largest_cut(X, W):
    """Bound of what the 8-bit matrix unit cuts off: of each product up to 2^-13 of the largest of its eight, itself
    whole; no more than 7 * 2^-13 of the sum of magnitudes."""
    return 7 * 2.0 ** -13 * (np.abs(X) @ np.abs(W).T)


@pytest.mark.parametrize("tokens,cols,rows", [s for s in SHAPES if s[1] >= 128])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_project_ordinary(backend, tokens, cols, rows, type):
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.ordinary(rng, tokens, cols, 1), p.ordinary(rng, rows, cols, 128)
    got, _ = product(backend, X, W, tokens, cols, rows, type, rows, 0)
    want = X[2] @ W[2].T
    # f32: at most 128 additions in a block, one a block after it and one a wave, each off by a step (2^-23) at most of a
    # partial sum, which the magnitudes' sum bounds
    sums = (128 + p.blocks(cols, 128) + 8) * 2.0 ** -23 * (np.abs(X[2]) @ np.abs(W[2]).T)
    bound = sums if type == "f32" else sums + largest_cut(X[2], W[2]) + 2.0 ** -8 * np.abs(want)
    assert np.all(np.abs(got - want) <= bound)
    # and on the whole: 80 roundings (four instructions a block, 20 blocks) to f32 at random are 9 * 2^-24 = 5e-7 of an
    # output's size, and 2e-6 allows four times that; 2^-9 / sqrt(3) is what rounding to bf16 costs
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= (2e-6 if type == "f32" else 2.0 ** -8)


@pytest.mark.parametrize("tokens,rows", [(3, 40), (300, 300)])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_project_special(backend, tokens, rows, type):
    """A NaN code poisons its token's or its row's outputs and no others; scales at both ends of the range."""
    cols = 300
    rng = np.random.default_rng(3)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    X[0][1, 7] = 0x7f
    W[0][33, 290] = 0xff
    X[1][2, 0] = 7     # 2^-120
    X[1][0, :] = 245   # 2^118
    W[1][:, 0], W[1][:, 1:] = 247, 0   # 2^120 and 2^-127
    got, _ = product(backend, X, W, tokens, cols, rows, type, rows, 0)
    with np.errstate(invalid="ignore", over="ignore"):
        x, w = p.values(X[0], X[1], 1), p.values(W[0], W[1], 128)
        want = np.array([[float((a * b).sum()) for b in w] for a in x[:3]])
    nan = np.isnan(got)
    assert nan[1].all() and nan[:, 33].all()
    ok = np.delete(np.arange(rows), 33)
    assert not nan[2:][:, ok].any()
    # token 0: sums at 2^238, their parts pass f32's range: not finite
    first = p.CODES[X[0][0, :128]] @ p.CODES[W[0][:, :128]].T
    assert not np.isfinite(got[0, ok])[first[ok] != 0].any()
    # token 2: 2^-120 * 2^120 = 1 beside products below 2^-110
    assert np.allclose(got[2, ok], want[2, ok], rtol=2.0 ** -8 if type == "bf16" else 2.0 ** -22, atol=1e-30)


def test_project_repeats(backend):
    """The same bits every time, and in a batch the bits do not depend on the other tokens."""
    rng = np.random.default_rng(9)
    X, W = p.ordinary(rng, 700, 2560, 1), p.ordinary(rng, 640, 2560, 128)
    for type in ("f32", "bf16"):
        a, _ = product(backend, X, W, 700, 2560, 640, type, 640, 0)
        b, _ = product(backend, X, W, 700, 2560, 640, type, 640, 0)
        assert np.array_equal(a, b)


# ------------------------------------------------------------------- gate_up
@pytest.mark.parametrize("tokens,cols,ff", [s for s in SHAPES if s[0] * s[2] < 4_000_000])
def test_gate_up(backend, tokens, cols, ff):
    """Exact sums, so that what is left is SiLU's f32 arithmetic: exp (one step), the sum, the quotient, the product."""
    rng = np.random.default_rng(tokens + cols + ff)
    X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    Wg[1][:] -= 5  # gates of about 1
    out = F8(backend, tokens, ff)
    ws = put(backend, np.full(backend.f8_gate_up_workspace_bytes(tokens, ff), 0xAA, np.uint8))
    backend.f8_gate_up(put(backend, X[0]), put(backend, X[1]), tokens, cols, put(backend, Wg[0]), put(backend, Wg[1]),
                       put(backend, Wu[0]), put(backend, Wu[1]), ff, out.codes, out.scales, ws)
    g, u = X[2] @ Wg[2].T / 32, X[2] @ Wu[2].T
    p.check_f8(*out.read(), p.silu(g) * u, 8 * HALF24)


def gate_up(be, X, Wg, Wu, tokens, cols, ff):
    out = F8(be, tokens, ff)
    ws = put(be, np.full(be.f8_gate_up_workspace_bytes(tokens, ff), 0xAA, np.uint8))
    be.f8_gate_up(put(be, X[0]), put(be, X[1]), tokens, cols, put(be, Wg[0]), put(be, Wg[1]), put(be, Wu[0]), put(be, Wu[1]),
                  ff, out.codes, out.scales, ws)
    return out.read()


# 128-token tiles in one round; 256-token tiles in one round, and in two of an even number of steps; a hidden size that
# ends inside a tile and its block (test_gpu_f8_tiles.py has the other rounds and steps)
FUSED = [(2000, 300, 2000), (1990, 512, 4000), (4000, 900, 3990)]


@pytest.mark.parametrize("tokens,cols,ff", FUSED)
def test_gate_up_many(backend, tokens, cols, ff):
    rng = np.random.default_rng(tokens + cols + ff)
    X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    Wg[1][:] -= 5
    g, u = (X[2].astype(np.float32) @ w[2].astype(np.float32).T for w in (Wg, Wu))  # exact
    p.check_f8(*gate_up(backend, X, Wg, Wu, tokens, cols, ff), p.silu(g.astype(np.float64) / 32) * u, 8 * HALF24)


@pytest.mark.parametrize("tokens,cols,ff", [(300, 640, 1000), (2000, 640, 2000), (4000, 1000, 3990)])
def test_gate_up_scales(backend, tokens, cols, ff):
    """The scales are those of the exact sums, where the matrix unit's are off by 1e-4: every eighth activation is large,
    so that the seven beside it lose their last bits. Blocks whose largest value lies within 1e-6 of a border are free."""
    rng = np.random.default_rng(tokens)
    x = rng.normal(0, 1, (tokens, cols))
    x[:, ::8] *= 40
    v, scales = p.quantize(x, 1)
    X = p.of_values(v, scales, 1, cols)
    Wg, Wu = p.ordinary(rng, ff, cols, 128), p.ordinary(rng, ff, cols, 128)
    for w in (Wg, Wu):
        w[1][:] -= 9
    codes, got = gate_up(backend, X, Wg, Wu, tokens, cols, ff)
    want = p.silu(X[2] @ Wg[2].T / 512) * (X[2] @ Wu[2].T / 512)
    amax = np.abs(p.padded(want, 1)).max((1, 3))
    kb = amax.shape[1]
    border = p.scale_exponents(amax * (1 - 1e-6)) != p.scale_exponents(amax * (1 + 1e-6))
    assert border.mean() < 1e-3
    assert np.array_equal(got[:, :kb][~border].astype(int) - 127, p.scale_exponents(amax)[~border])
    assert np.linalg.norm(p.values(codes, got, 1)[:, :ff] - want) / np.linalg.norm(want) < 0.03


@pytest.mark.parametrize("tokens,ff", [(128, 256), (2000, 2000)])
def test_gate_up_silu(backend, tokens, ff):
    """One product a sum: gates of every e4m3 value up to 224 and, in half the tokens, only far below 0, where silu is as
    small as 1e-33; u = 1."""
    cols = 128
    rng = np.random.default_rng(tokens)
    X, W, U = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    X[0][:], X[1][:] = 0, 127
    X[0][np.arange(tokens), np.arange(tokens) % cols] = 0x38  # 1
    W[0][:] = rng.integers(0, 256, W[0].shape)
    W[0][(W[0] & 127) == 127] = 0
    W[1][:] = 126
    W[0][:, 1::2] = 0xef + rng.integers(0, 4, (ff, cols // 2))  # -60, -64, -72, -80
    U[0][:], U[1][:] = 0x38, 127
    codes, scales = gate_up(backend, X, W, U, tokens, cols, ff)
    g = p.CODES[W[0][:, np.arange(tokens) % cols]].T / 2
    assert g[1::2].max() <= -56 and g.max() == 224 and g.min() == -224
    p.check_f8(codes, scales, g / (1 + np.exp(-g)), 8 * HALF24)


@pytest.mark.parametrize("tokens,cols,ff", [(3, 300, 200), (100, 300, 200), (2000, 300, 2000)])
def test_gate_up_special(backend, tokens, cols, ff):
    """A NaN among a token's codes makes its outputs NaN, one in a row of weights that column's; the others, and the
    scales, go by what is finite."""
    rng = np.random.default_rng(3)
    X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    Wg[1][:] -= 5
    X[0][1, 7], Wg[0][33, 290], Wu[0][130, 0] = 0x7f, 0xff, 0x7f
    codes, scales = gate_up(backend, X, Wg, Wu, tokens, cols, ff)
    got = p.CODES[codes][:, :ff]
    bad = np.zeros((tokens, ff), bool)
    bad[1] = bad[:, 33] = bad[:, 130] = True
    assert np.array_equal(np.isnan(got), bad)
    assert np.all(scales[1] == 127)
    want = p.silu(X[2] @ Wg[2].T / 32) * (X[2] @ Wu[2].T)
    want[bad] = 0
    codes = codes.copy()
    codes[:, :ff][bad] = 0
    p.check_f8(codes, scales, want, 8 * HALF24)


@pytest.mark.parametrize("tokens,cols,ff", [(1, 2560, 640), (40, 700, 513), (130, 1024, 400), (400, 2560, 640)])
def test_gate_up_ordinary(backend, tokens, cols, ff):
    rng = np.random.default_rng(tokens + cols + ff)
    X, Wg, Wu = p.ordinary(rng, tokens, cols, 1), p.ordinary(rng, ff, cols, 128), p.ordinary(rng, ff, cols, 128)
    for w in (Wg, Wu):
        w[1][:] -= 6
    out = F8(backend, tokens, ff)
    ws = put(backend, np.zeros(backend.f8_gate_up_workspace_bytes(tokens, ff), np.uint8))
    backend.f8_gate_up(put(backend, X[0]), put(backend, X[1]), tokens, cols, put(backend, Wg[0]), put(backend, Wg[1]),
                       put(backend, Wu[0]), put(backend, Wu[1]), ff, out.codes, out.scales, ws)
    codes, scales = out.read()
    want = p.silu(X[2] @ Wg[2].T / 64) * (X[2] @ Wu[2].T / 64)
    got = p.values(codes, scales, 1)[:, :ff]
    # rounding to 4 significant bits: 2^-4 at most, 2^-4 / sqrt(12) * sqrt(8/7...) on the whole, under 0.03
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 0.03


# -------------------------------------------------------------- run together
def feed_forward(be, tokens, width, ff, b, x, r):
    """h = x + r; y = h + down(silu(gate(norm(h))) * up(norm(h))) in one buffer."""
    be.f8_norm(x, b["gamma"], 1e-6, tokens, width, b["n"].codes, b["n"].scales, residual=r, H=b["h"])
    be.f8_gate_up(b["n"].codes, b["n"].scales, tokens, width, b["wg"].codes, b["wg"].scales, b["wu"].codes, b["wu"].scales,
                  ff, b["a"].codes, b["a"].scales, b["ws"])
    be.f8_project(b["a"].codes, b["a"].scales, tokens, ff, b["wd"].codes, b["wd"].scales, width, b["h"], residual=b["h"])


@pytest.mark.parametrize("tokens,width,ff", [(1, 640, 1000), (37, 256, 384), (300, 640, 1000)])
def test_feed_forward_block(backend, tokens, width, ff):
    """A block from f32 weights and activations, called and replayed from a graph with eager calls between, against
    the same steps in 64 bits from the GPU's own codes, and near the block without 8 bits."""
    be = backend
    rng = np.random.default_rng(tokens)
    w = {k: rng.normal(0, s ** -0.5, shape).astype(np.float32)
         for k, shape, s in (("wg", (ff, width), width), ("wu", (ff, width), width), ("wd", (width, ff), ff))}
    gamma = rng.normal(1, 0.1, width).astype(np.float32)
    x, r = (rng.normal(0, 1, (tokens, width)).astype(np.float32) for _ in range(2))
    b = {"gamma": put(be, gamma), "n": F8(be, tokens, width), "a": F8(be, tokens, ff),
         "h": put(be, np.zeros((tokens, width), np.float32)),
         "ws": be.alloc_bytes(be.f8_gate_up_workspace_bytes(tokens, ff))}
    for k, v in w.items():
        b[k] = F8(be, *v.shape, 128)
        be.f8_quantize(put(be, v), *v.shape, 128, b[k].codes, b[k].scales)
    X, R = put(be, x), put(be, r)
    feed_forward(be, tokens, width, ff, b, X, R)
    y = get(be, b["h"], np.float32, (tokens, width))
    h = (x + r).astype(np.float64)
    codes, scales = b["n"].read()
    p.check_f8(codes, scales, h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6) * gamma, 4 * HALF24)
    n, a = p.values(codes, scales, 1)[:, :width], p.values(*b["a"].read(), 1)[:, :ff]
    wv = {k: p.values(*b[k].read(), 128)[:, :v.shape[1]] for k, v in w.items()}
    act = p.silu(n @ wv["wg"].T) * (n @ wv["wu"].T)
    assert np.linalg.norm(a - act) / np.linalg.norm(act) < 0.03
    want = h + a @ wv["wd"].T
    mag = np.abs(h) + np.abs(a) @ np.abs(wv["wd"]).T
    assert np.all(np.abs(y - want) <= (128 + p.blocks(ff, 128) + 9) * 2.0 ** -23 * mag)
    plain = h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6) * gamma
    plain = h + (p.silu(plain @ w["wg"].T) * (plain @ w["wu"].T)) @ w["wd"].T
    assert np.linalg.norm(y - plain) / np.linalg.norm(plain - h) < 0.1

    be.idle()
    be.graph_begin()
    feed_forward(be, tokens, width, ff, b, X, R)
    graph = be.graph_end()
    for k in range(4):  # other inputs, eager work and a wait between the replays
        x2 = np.roll(x, k, 1)
        be.write(X, x2)
        be.graph_launch(graph)
        replayed = get(be, b["h"], np.float32, (tokens, width))
        feed_forward(be, tokens, width, ff, b, X, R)
        assert np.array_equal(get(be, b["h"], np.float32, (tokens, width)), replayed)
        if k == 0:
            assert np.array_equal(replayed, y)
    be.graph_free(graph)


def test_two_graphs_share_a_workspace(backend):
    """Two captured gated pairs of one workspace run in turn."""
    be, tokens, cols, ff = backend, 20, 256, 512
    rng = np.random.default_rng(1)
    ws = be.alloc_bytes(be.f8_gate_up_workspace_bytes(tokens, ff))
    graphs, outs = [], []
    for _ in range(2):
        X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
        Wg[1][:] -= 5
        bufs = [put(be, a) for m in (X, Wg, Wu) for a in m[:2]]
        out = F8(be, tokens, ff)
        be.idle()
        be.graph_begin()
        be.f8_gate_up(bufs[0], bufs[1], tokens, cols, *bufs[2:], ff, out.codes, out.scales, ws)
        graphs.append(be.graph_end())
        outs.append((out, p.silu(X[2] @ Wg[2].T / 32) * (X[2] @ Wu[2].T)))
    for _ in range(3):
        for g in graphs:
            be.graph_launch(g)
    for out, want in outs:
        p.check_f8(*out.read(), want, 8 * HALF24)
    for g in graphs:
        be.graph_free(g)


def test_two_contexts(backend):
    """Calls of two contexts, on their own streams, under way together."""
    import stratacuda_amd as sm
    rng = np.random.default_rng(2)
    other = sm.Backend(0)
    try:
        shapes = [(backend, 900, 700, 1500), (other, 400, 1300, 2100)]
        runs = []
        for be, tokens, cols, rows in shapes:
            X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
            bufs = [put(be, a) for a in (X[0], X[1], W[0], W[1])]
            runs.append((be, tokens, cols, rows, bufs, put(be, np.zeros((tokens, rows), np.float32)),
                         (X[2] @ W[2].T).astype(np.float32)))
        for _ in range(20):
            for be, tokens, cols, rows, b, Y, _ in runs:
                be.f8_project(b[0], b[1], tokens, cols, b[2], b[3], rows, Y)
        for be, tokens, cols, rows, b, Y, want in runs:
            assert np.array_equal(get(be, Y, np.float32, (tokens, rows)), want)
    finally:
        other.dispose()


# ----------------------------------------- products whose waves share out the columns
STREAMS = [  # tokens, cols, rows: workgroups of (tokens x rows; to f32, to bf16, gated), the last ones ending inside
    (5, 2570, 4003),    # 16 x 16
    (2003, 260, 20),    # the same, tokens over the XCDs, fewer blocks than waves
    (19, 1300, 2505),   # 32 x 16
    (70, 1290, 2503),   # 32 x 32 (gated 32 x 16)
    (17, 2500, 5003),   # gated 32 x 32
    (97, 1300, 2503),   # 64 x 32
    (131, 260, 5003),   # 32 x 64 (to bf16 tiles of 64 x 64, gated 64 x 32)
    (3, 6010, 10003),   # to bf16 32 x 64 (the others 16 x 16)
    (205, 2600, 2503)]  # 64 x 64 (gated 64 x 32)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("extra,offset", [(3, 2), (5, 4)])
@pytest.mark.parametrize("tokens,cols,rows", STREAMS)
def test_project_streams(backend, tokens, cols, rows, type, extra, offset):
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    got, rest = product(backend, X, W, tokens, cols, rows, type, rows + extra, offset)
    want = X[2].astype(np.float32) @ W[2].astype(np.float32).T  # exact in f32: every partial sum is
    assert np.array_equal(got, want if type == "f32" else p.bf16(want).astype(np.float32))
    assert np.all(rest == -7)


@pytest.mark.parametrize("tokens,cols,rows", STREAMS)
def test_project_streams_residual(backend, tokens, cols, rows):
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    r = rng.normal(0, 100, tokens * rows + 3).astype(np.float32)
    Y = put(backend, r)
    got, rest = product(backend, X, W, tokens, cols, rows, "f32", rows, 0, residual=Y, Y=Y)
    assert np.array_equal(got, r[:-3].reshape(tokens, rows) + X[2].astype(np.float32) @ W[2].astype(np.float32).T)
    assert np.array_equal(rest, r[-3:])


@pytest.mark.parametrize("tokens,cols,ff", STREAMS)
def test_gate_up_streams(backend, tokens, cols, ff):
    rng = np.random.default_rng(tokens + cols + ff)
    X, Wg, Wu = p.matrix(rng, tokens, cols, 1), p.matrix(rng, ff, cols, 128), p.matrix(rng, ff, cols, 128)
    Wg[1][:] -= 5
    g, u = (X[2].astype(np.float32) @ w[2].astype(np.float32).T for w in (Wg, Wu))  # exact
    p.check_f8(*gate_up(backend, X, Wg, Wu, tokens, cols, ff), p.silu(g.astype(np.float64) / 32) * u, 8 * HALF24)


@pytest.mark.parametrize("tokens,cols,rows", [(3, 6010, 10003), (97, 1300, 2503), (205, 2600, 2503)])
def test_project_streams_nan(backend, tokens, cols, rows):
    """A NaN code of the last token and one of the last row, in the last block: no other output sees them."""
    rng = np.random.default_rng(rows)
    X, W = p.matrix(rng, tokens, cols, 1), p.matrix(rng, rows, cols, 128)
    X[0][tokens - 1, cols - 1] = 0x7f
    W[0][rows - 1, cols - 1] = 0xff
    for type in ("f32", "bf16"):
        got, _ = product(backend, X, W, tokens, cols, rows, type, rows, 0)
        nan = np.isnan(got)
        assert nan[-1].all() and nan[:, -1].all() and not nan[:-1, :-1].any()


@pytest.mark.parametrize("tokens,cols,rows", [(17, 2500, 5003), (97, 1300, 2503), (205, 2600, 2503)])
def test_project_streams_ordinary(backend, tokens, cols, rows):
    rng = np.random.default_rng(tokens + cols + rows)
    X, W = p.ordinary(rng, tokens, cols, 1), p.ordinary(rng, rows, cols, 128)
    want, size = X[2] @ W[2].T, np.abs(X[2]) @ np.abs(W[2]).T
    for type in ("f32", "bf16"):
        got, _ = product(backend, X, W, tokens, cols, rows, type, rows, 0)
        # as in test_project_ordinary: 128 additions in a block, one a block, one a wave
        sums = (128 + p.blocks(cols, 128) + 8) * 2.0 ** -23 * size
        assert np.all(np.abs(got - want) <= (sums if type == "f32" else sums + largest_cut(X[2], W[2]) + 2.0 ** -8 * np.abs(want)))
