"""Comparison of results of attention over a 4-bit cache with 64 bits in which
what is no number fails. No counterpart in the reference."""
import numpy as np

import kv4_plain as plain

LOG2E = 1.4426950408889634


def outside(got, want, off):
    """Where `got` is not within `off` of `want`: a NaN on either side, or in `off`, is nowhere within."""
    with np.errstate(invalid="ignore"):
        return ~(np.abs(got - want) <= off)


def limit(size, y, length, exponent, type):
    """How far a result may be off: `size` is the sum of p |v| over l, `exponent` the largest exponent in powers of two. A
    probability is off by its exponent's rounding and by the exponential's, 2^-22 of the exponent's size and of itself, twice for
    a sum brought to another maximum; the sums of up to `length` positions by 2^-23 each, above and below. bf16 adds half a step,
    2^-9 of a number between two powers of two and at most 2^-8, for the probability and for the result."""
    off = size * (2.0 ** -21 * (2 + exponent) + (length + 64) * 2.0 ** -22)
    return off + (2.0 ** -8 * (size + np.abs(y)) if type == "bf16" else 0) + 1e-30


def expect(b, q, got, scale, type, window=0, gate=None, fill=9.0, left=(), most=1 << 30):
    """Every row of batch b against 64 bits, of sequences of more than `most` rows that many, the first and last ones among them,
    the others for being numbers; the rows of the sequences `left`, and those of none, as they were."""
    for s, (n, length) in enumerate(b.sequences):
        a = b.starts[s]
        if s in left:
            assert np.all(got[a:a + n] == fill), s
            continue
        k, v = b.held(s)
        assert np.isfinite(got[a:a + n]).all(), s
        at = np.unique(np.linspace(0, n - 1, min(n, most)).astype(int)) if n else np.arange(0)
        y, size = plain.attention(q[a + at].astype(np.float64), length - n + at, k, v, scale, window,
                                  None if gate is None else gate[a + at].astype(np.float64))
        exponent = scale * LOG2E * np.abs(q).max() * (np.abs(k).sum(-1).max() if k.size else 0)
        bad = outside(got[a + at], y, limit(size, y, length, exponent, type))
        assert not bad.any(), (s, int(bad.sum()), np.argwhere(bad)[:4], got[a + at][bad][:4], y[bad][:4])
    assert np.all(got[b.rows:] == fill)
