"""Attention over a 4-bit cache where scores are far from 0, up to f32's range,
against 64 bits. Queries and codes are those whose scores are exact, multiples
of 2^-4 before the scale, of at least 2^12 here: the probability of a score
that is not the row's largest is below e^-256, and those of n that are it 1/n.
Scores of one row cancel in whatever is lost of their common size, so that the
bound of a score of 0 holds (kv4_compare). No counterpart in the reference."""
import numpy as np
import pytest

import kv4_batches as batches
import kv4_plain as plain
from kv4_compare import limit, outside
from test_gpu_kv4 import Batch, queries, run_attention

pytestmark = pytest.mark.gpu
SCALES = [2.0 ** 12, 1.3 * 2.0 ** 17, 2.0 ** 18, 1.9 * 2.0 ** 18, 1.3 * 2.0 ** 20, 2.0 ** 21, 2.0 ** 30, 1.1 * 2.0 ** 64, 2.0 ** 99]


@pytest.fixture(scope="module")
def be(backend):
    yield backend


def copy_key(tiles, page, at, from_page, from_at):
    """The key of one position to another, in all heads."""
    pitch = tiles.shape[-1] // 68
    to, of = tiles[page], tiles[from_page]
    to[:, at * pitch // 2:(at + 1) * pitch // 2] = of[:, from_at * pitch // 2:(from_at + 1) * pitch // 2]
    for b in range(pitch // 32):
        to[:, 64 * pitch + b * 64 + at % 16 * 4 + at // 16] = of[:, 64 * pitch + b * 64 + from_at % 16 * 4 + from_at // 16]


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 256), ("f32", 64), ("f32", 128)])
@pytest.mark.parametrize("name,sign", [("WHOLE", "both"), ("WHOLE", "below"), ("WHOLE", "above"), ("PIECES", "both"), ("PIECES", "below"),
                                       ("FEW", "both"), ("FEW", "below"), ("FEW", "above"), ("MIXED", "both")])
def test_far_scores(be, name, sign, type, dim):
    rng = np.random.default_rng(dim)
    which = getattr(batches, name)
    b = Batch(be, rng, which["sequences"], which["kv"], dim, extra_rows=1, table_pages=which["width"])
    q = queries(rng, (b.tokens, which["heads"], dim))
    if sign != "both":  # keys of one sign, queries of the other one or the same
        pitch = plain.pitch_of(dim)
        b.host.reshape(-1, 68 * pitch)[:, :32 * pitch] |= 0x88
        b.clear_padding()
        q = np.abs(q) if sign == "below" else -np.abs(q)
    there = [s for s, (n, length) in enumerate(b.sequences) if n and length]
    some = sorted(set(there[:2] + sorted(there, key=lambda s: -b.sequences[s][0])[:2]))
    tiles = b.host.reshape(-1, b.kv, 68 * plain.pitch_of(dim))
    for s in some:  # positions in threes have one key: rows of one, two or three largest scores
        for p in range(b.sequences[s][1]):
            copy_key(tiles, b.page(s, p), p % 64, b.page(s, p - p % 3), (p - p % 3) % 64)
    held = {s: b.held(s) for s in some}
    b.upload()
    for scale in np.float32(SCALES):
        got = run_attention(be, b, q, float(scale), type)
        for s in some:
            n, length = b.sequences[s]
            at = np.unique(np.linspace(0, n - 1, 6).astype(int))
            rows = b.starts[s] + at
            y, size = plain.attention(q[rows].astype(np.float64), length - n + at, *held[s], float(scale))
            bad = outside(got[rows], y, limit(size, y, length, 0, type))
            assert not bad.any(), (float(scale), s, int(bad.sum()), got[rows][bad][:4], y[bad][:4])
    b.free()
