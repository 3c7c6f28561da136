"""Attention over a 4-bit cache where windows are large, tables are wider than
their contexts and rows lie before position 0, against 64 bits (kv4_compare).
Queries and codes are those whose scores are exact. No counterpart in the
reference."""
import numpy as np
import pytest

import kv4_batches as batches
import kv4_plain as plain
from kv4_compare import expect
from test_gpu_kv4 import Batch, queries, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(backend):
    yield backend


# The batches of kv4_batches with rows before position 0 in sequences of both ends of a workgroup's search.
BEFORE = {
    "WHOLE": dict(batches.WHOLE, sequences=[(70, 40), (130, 3), (1, 129), (33, 33), (3, 3)] + [(0, 9)] * 19),
    "PIECES": dict(batches.PIECES, sequences=[(17, 1500), (130, 70), (5, 0), (1, 64), (96, 95), (2, 130)]),
    "FEW": dict(batches.FEW, sequences=[(1, 1500), (3, 1), (2, 0), (1, 64), (3, 2)]),
    "SOME": dict(batches.SOME, sequences=[(20, 15), (16, 700), (5, 0), (1, 64)]),
}


def before(be, rng, name, dim):
    which = BEFORE[name]
    return which, Batch(be, rng, which["sequences"], which["kv"], dim, extra_rows=2, table_pages=which["width"])


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 128)])
@pytest.mark.parametrize("name", BEFORE)
def test_a_window_past_every_position_is_none(be, name, type, dim):
    rng = np.random.default_rng(dim)
    which, b = before(be, rng, name, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    none = run_attention(be, b, q, scale, type)
    expect(b, q, none, scale, type)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 100, 2 ** 30, 64 * which["width"]):
        wrong = (run_attention(be, b, q, scale, type, window=window) != none).any((1, 2))
        assert not wrong.any(), (window, np.flatnonzero(wrong)[:8])
    # a position less: the first one is still every row's, but the kernels ask
    window = 64 * which["width"] - 1
    expect(b, q, run_attention(be, b, q, scale, type, window=window), scale, type, window=window)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 200), ("f32", 128)])
@pytest.mark.parametrize("name", BEFORE)
@pytest.mark.parametrize("window", [1, 2, 64, 100, 600])
def test_a_window_and_rows_before_position_0(be, window, name, type, dim):
    rng = np.random.default_rng(dim + window)
    which, b = before(be, rng, name, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    expect(b, q, run_attention(be, b, q, scale, type, window=window), scale, type, window=window)
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_read_heads_first(be, type):
    """Keys and values as an array of heads has them, each head's rows together."""
    rng = np.random.default_rng(3)
    kv, dim = 3, 72
    b = Batch(be, rng, [(70, 130), (5, 3), (1, 64)], kv, dim, extra_rows=1)
    n = b.tokens
    K, V = (be.alloc(plain.bits(np.full(n * kv * dim + 8, 7, np.float32), type)) for _ in range(2))
    be.kv4_read(b.pool, b.pages, kv, dim, b.seqs, K, V, k_view=(dim, n * dim, 8), v_view=(dim, n * dim, 0), type=type)
    for buf, which, offset in ((K, 0, 8), (V, 1, 0)):
        got = plain.from_bits(be.read_bytes(buf), type)[offset:offset + n * kv * dim].reshape(kv, n, dim)
        for s, (rows, length) in enumerate(b.sequences):
            for i in range(rows):
                p = length - rows + i
                want = plain.get(b.host, kv, dim, b.page(s, p), p % 64)[which] if p >= 0 else np.zeros((kv, dim))
                assert np.array_equal(got[:, b.starts[s] + i], want), (s, i)
        assert np.all(got[:, b.rows:] == 7)
        be.free(buf)
    b.free()
