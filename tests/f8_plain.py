"""The 8-bit floating-point operators in 64 bits with numpy, from their
definitions: e4m3 values by rounding to nearest even, power-of-two scales, sums
of products. No counterpart in the reference."""
import numpy as np

TOP = 448.0
HALF24 = 2.0 ** -24  # half a step of f32, relative


def _code_values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10), m * 2.0 ** -9)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


CODES = _code_values()


def step(v):
    """The distance between e4m3 values around v."""
    e = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -9)))
    return 2.0 ** (np.maximum(e, -6) - 3)


def round_e4m3(v):
    v = np.asarray(v, np.float64)
    m, e = np.frexp(v)
    s = 2.0 ** (np.maximum(e, -5) - 4.0)
    return np.rint(v / s) * s


def blocks(n, block):
    return -(-n // block)


def layout(rows, cols, block):
    """(pitch, scale pitch, rows of scales)"""
    kb = blocks(cols, 128)
    return kb * 128, 4 * blocks(kb, 4), blocks(rows, block)


def padded(x, block):
    """x as [row blocks, block, column blocks, 128] in f64, zeros past its edges."""
    rows, cols = x.shape
    pitch, _, up = layout(rows, cols, block)
    p = np.zeros((up * block, pitch))
    p[:rows, :cols] = x
    return p.reshape(up, block, pitch // 128, 128)


def scale_exponents(amax):
    """The smallest e >= -127 with amax <= 448 * 2^e, 0 for amax = 0."""
    e = np.full(amax.shape, -127)
    while True:
        low = (amax > TOP * 2.0 ** e.astype(np.float64))
        if not low.any():
            return np.where(amax > 0, e, 0)
        e = e + low


def quantize(x, block):
    """(code values [rows, pitch] with NaN where x is not finite, scale bytes [row blocks, scale pitch])"""
    rows, cols = x.shape
    pitch, spitch, up = layout(rows, cols, block)
    b = padded(x, block)
    e = scale_exponents(np.where(np.isfinite(b), np.abs(b), 0.0).max((1, 3)))
    v = np.where(np.isfinite(b), b, np.nan) * 2.0 ** -e[:, None, :, None].astype(np.float64)
    scales = np.full((up, spitch), 127, np.uint8)
    scales[:, : pitch // 128] = e + 127
    return round_e4m3(v).reshape(up * block, pitch)[:rows], scales


def values(codes, scales, block):
    """The matrix that code bytes [rows, pitch] and scale bytes stand for, columns past the edge included."""
    rows, pitch = codes.shape
    s = 2.0 ** (scales[:, : pitch // 128].astype(np.float64) - 127)
    return CODES[codes] * s.repeat(block, 0)[:rows].repeat(128, 1)


def bf16(x):
    """x rounded to bf16 (nearest even), in f64; x must lie well inside f32's range."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.rint(m * 256.0) / 256.0, e)


def bf16_bits(x):
    return (np.ascontiguousarray(bf16(x), np.float32).view(np.uint32) >> 16).astype(np.uint16)


def from_bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def check_f8(codes, scales, y, off, block=1):
    """Codes and scale bytes are y's up to a relative error `off` of y before the rounding: each
    block's scale the smallest that holds its largest value, each code within half a step (and
    `off`) of y over the scale, codes past the edge 0 and scales past it 127."""
    rows, cols = y.shape
    pitch, spitch, up = layout(rows, cols, block)
    assert codes.shape == (rows, pitch) and scales.shape == (up, spitch)
    kb = pitch // 128
    assert np.all(scales[:, kb:] == 127)
    b = padded(y, block)
    amax = np.abs(b).max((1, 3))
    s = 2.0 ** (scales[:, :kb].astype(np.float64) - 127)
    zero = amax == 0
    assert np.all(s[zero] == 1)
    assert np.all((amax <= TOP * s * (1 + off))[~zero])
    assert np.all((amax * (1 + off) >= TOP * s / 2)[~zero] | (s[~zero] == 2.0 ** -127))
    each = s.repeat(block, 0)[:rows].repeat(128, 1)
    want = b.reshape(up * block, pitch)[:rows] / each
    got = CODES[codes]
    bad = np.abs(got - want) > step(want * (1 + off)) / 2 + np.abs(want) * off
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])
    assert np.all(codes[:, cols:] & 127 == 0)


def matrix(rng, rows, cols, block):
    """A matrix whose products and sums are exact in any order: code values from {0, +-1/2, +-1, +-2} and scales 2^-2 to 2^2.
    (code bytes, scale bytes, the values in f64 [rows, cols])"""
    pitch, spitch, up = layout(rows, cols, block)
    table = np.array([0x00, 0x30, 0x38, 0x40, 0xb0, 0xb8, 0xc0], np.uint8)
    codes = np.zeros((rows, pitch), np.uint8)
    codes[:, :cols] = table[rng.integers(0, 7, (rows, cols))]
    scales = np.full((up, spitch), 127, np.uint8)
    scales[:, : pitch // 128] = rng.integers(125, 130, (up, pitch // 128))
    return codes, scales, values(codes, scales, block)[:, :cols]


def of_values(v, scales, block, cols):
    """(code bytes, scale bytes, the matrix) of code values [rows, pitch]."""
    order = np.argsort(CODES[:127])
    at = np.searchsorted(CODES[:127][order], np.abs(v))
    codes = (order[at] | np.where(np.signbit(v), 128, 0)).astype(np.uint8)
    return codes, scales, values(codes, scales, block)[:, :cols]


def ordinary(rng, rows, cols, block):
    """The same as matrix() of normal values, some columns larger."""
    x = rng.normal(0, 1, (rows, cols)) * np.exp(rng.normal(0, 0.8, cols))
    return of_values(*quantize(x, block), block, cols)


def silu(g):
    return g / (1 + np.exp(-g))
