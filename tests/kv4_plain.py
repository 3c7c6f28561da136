"""Attention over a 4-bit key-value cache in 64 bits with numpy, from the
operators' definitions. No counterpart in the reference."""
import numpy as np

PAGE = 64
CODES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def pitch_of(dim):
    return -(-dim // 64) * 64


def page_bytes(kv, dim):
    return kv * 68 * pitch_of(dim)


def scale_bytes(amax):
    """The byte of the smallest 2^e, -125 <= e <= 125, with amax <= 6 * 2^e; 127 for 0, 255 where amax is not finite."""
    e = np.full(amax.shape, -125)
    while True:
        low = np.isfinite(amax) & (amax > 6 * 2.0 ** e) & (e < 125)
        if not low.any():
            return np.where(np.isfinite(amax), np.where(amax > 0, e + 127, 127), 255).astype(np.uint8)
        e = e + low


def quantize(x):
    """(codes [.., pitch], scale bytes [.., pitch / 32]) of x [.., dim], the nearest code by comparison, ties to the even one."""
    dim = x.shape[-1]
    b = np.zeros(x.shape[:-1] + (pitch_of(dim),))
    b[..., :dim] = x
    b = b.reshape(b.shape[:-1] + (-1, 32))
    with np.errstate(invalid="ignore"):
        amax = np.where(np.isnan(b).any(-1), np.nan, np.abs(b).max(-1))
    scales = scale_bytes(amax)
    bad = scales == 255
    b = np.where(bad[..., None], 0.0, b)
    y = np.abs(b) / np.where(bad, 1.0, 2.0 ** (scales.astype(np.float64) - 127))[..., None]
    distance = np.abs(y[..., None] - CODES[:8])
    even = distance + np.array([0, 1, 0, 1, 0, 1, 0, 1]) * 1e-9  # among equals the even code
    codes = np.argmin(even, -1).astype(np.uint8)
    codes |= (np.signbit(b) << 3).astype(np.uint8)
    return codes.reshape(codes.shape[:-2] + (-1,)), scales


def numbers(codes, scales):
    """What codes [.., pitch] and scale bytes [.., pitch / 32] stand for."""
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return CODES[codes] * np.repeat(s, 32, -1)


def put(pool, kv, dim, page, at, k, v):
    """Keys and values [kv, dim] of one position into byte array `pool`, each byte where the layout has it."""
    pitch = pitch_of(dim)
    nb = pitch // 32
    g, q, i, n = at // 16, at // 4 % 4, at % 4, at % 16
    for h in range(kv):
        tile = pool[(page * kv + h) * 68 * pitch:][:68 * pitch]
        c, s = quantize(k[h])
        tile[at * pitch // 2:(at + 1) * pitch // 2] = c[0::2] | c[1::2] << 4
        c2, s2 = quantize(v[h])
        for b in range(nb):
            tile[64 * pitch + b * 64 + n * 4 + g] = s[b]
            tile[66 * pitch + b * 64 + q * 16 + g * 4 + i] = s2[b]
            for r in range(16):
                tile[32 * pitch + b * 1024 + (q * 16 + r) * 16 + g * 4 + i] = c2[32 * b + r] | c2[32 * b + 16 + r] << 4


def get(pool, kv, dim, page, at):
    """(keys, values) [kv, dim] of one position."""
    pitch = pitch_of(dim)
    nb = pitch // 32
    g, q, i, n = at // 16, at // 4 % 4, at % 4, at % 16
    keys, values = np.empty((kv, dim)), np.empty((kv, dim))
    b, r = np.arange(nb), np.arange(16)
    for h in range(kv):
        tile = pool[(page * kv + h) * 68 * pitch:][:68 * pitch]
        w = tile[at * pitch // 2:(at + 1) * pitch // 2]
        keys[h] = numbers(np.stack([w & 15, w >> 4], -1).reshape(-1), tile[64 * pitch + b * 64 + n * 4 + g])[:dim]
        w = tile[32 * pitch + b[:, None] * 1024 + (q * 16 + r) * 16 + g * 4 + i]
        values[h] = numbers(np.stack([w & 15, w >> 4], 1).reshape(-1), tile[66 * pitch + b * 64 + q * 16 + g * 4 + i])[:dim]
    return keys, values


def attention(q, positions, keys, values, scale, window=0, gate=None):
    """(y [n, heads, dim], the sum of p |v| over l of each) of rows at `positions`; keys, values [length, kv, dim], NaN rows in
    `keys` count as any; `there` positions only: pass those of a sequence in order. Rows without positions are 0."""
    n, heads, dim = q.shape
    kv = keys.shape[1]
    y, size = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    for i in range(n):
        hi = positions[i]
        lo = max(0, hi - window + 1) if window else 0
        if hi < 0:
            continue
        for h in range(heads):
            j = h // (heads // kv)
            s = scale * (keys[lo:hi + 1, j] @ q[i, h])
            p = np.exp(s - s.max())
            y[i, h] = (p[:, None] * values[lo:hi + 1, j]).sum(0) / p.sum()
            size[i, h] = (p[:, None] * np.abs(values[lo:hi + 1, j])).sum(0) / p.sum()
    if gate is not None:
        with np.errstate(over="ignore"):
            f = 1 / (1 + np.exp(-gate))
        y, size = y * f, size * f
    return y, size


def norm_rope(x, gamma, eps, cos, sin, rotary, positions):
    x = np.asarray(x, np.float64)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma
    half = rotary // 2
    c, s = cos[positions][:, None].astype(np.float64), sin[positions][:, None].astype(np.float64)
    y = n.copy()
    y[..., :half] = n[..., :half] * c - n[..., half:rotary] * s
    y[..., half:rotary] = n[..., half:rotary] * c + n[..., :half] * s
    return y, n


def bf16(x):
    """x rounded to bf16 (nearest even) as f32; x finite and well inside f32's range, or NaN."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.rint(m * 256.0) / 256.0, e).astype(np.float32)


def bits(x, type):
    """x as the library takes it: f32, or the bits of bf16."""
    x = np.ascontiguousarray(x, np.float32)
    return x if type == "f32" else (x.view(np.uint32) >> 16).astype(np.uint16)


def from_bits(raw, type):
    """f32 values of bytes."""
    if type == "f32":
        return raw.view(np.float32)
    return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32)
