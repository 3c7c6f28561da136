"""Attention over a 4-bit cache of batches whose sequences' rows differ, over
long contexts: each sequence's own tiles in pieces, against 64 bits
(kv4_compare). test_kv4_unlike.py holds the batches to that. No counterpart in
the reference."""
import numpy as np
import pytest

import kv4_batches as batches
import kv4_plain as plain
from kv4_compare import expect
from test_gpu_kv4 import Batch, queries, run_attention

pytestmark = pytest.mark.gpu
NAMES = ["UNLIKE", "UNLIKE_PROMPT"]


@pytest.fixture(scope="module")
def be(backend):
    yield backend


def batch(be, rng, name, dim, sequences=None, **more):
    which = getattr(batches, name)
    return which["heads"], Batch(be, rng, sequences or which["sequences"], which["kv"], dim, extra_rows=2, table_pages=which["width"], **more)


@pytest.mark.parametrize("type,dim", batches.TYPES)
@pytest.mark.parametrize("name", NAMES)
def test_attention(be, name, type, dim):
    rng = np.random.default_rng(dim)
    heads, b = batch(be, rng, name, dim)
    q, g = queries(rng, (b.tokens, heads, dim)), plain.bf16(rng.normal(0, 4, (b.tokens, heads, dim)))
    gv = (heads * dim + 5, dim, 1)
    scale = dim ** -0.5 / 8
    expect(b, q, run_attention(be, b, q, scale, type, gate=g, gate_view=gv), scale, type, gate=g, most=24)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("window", [1, 100, 2100, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("name", NAMES)
def test_window(be, name, window, type, dim):
    rng = np.random.default_rng(window)
    heads, b = batch(be, rng, name, dim)
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 8
    expect(b, q, run_attention(be, b, q, scale, type, window=window), scale, type, window=window, most=24)
    b.free()


@pytest.mark.parametrize("name", NAMES)
def test_more_sequences_than_a_wave(be, name):
    rng = np.random.default_rng(1)
    which = getattr(batches, name)
    sequences = [(1, 1 + 70 * i) if i % 3 else (0, 5) for i in range(75)] + [which["sequences"][1]]
    heads, b = batch(be, rng, name, 64, sequences)
    q = queries(rng, (b.tokens, heads, 64))
    expect(b, q, run_attention(be, b, q, 0.02, "bf16"), 0.02, "bf16", most=24)
    b.free()


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("name", NAMES)
def test_captured_and_replayed(be, name, type):
    """A graph takes the starts, lengths and tables that stand there when it runs; nothing past the workspace is written."""
    rng = np.random.default_rng(2)
    dim, scale = 64, 0.02
    heads, b = batch(be, rng, name, dim)
    q = queries(rng, (b.tokens, heads, dim))
    Q, Y = be.alloc(plain.bits(q, type)), be.alloc(plain.bits(np.zeros(q.size, np.float32), type))
    n = be.kv4_attention_workspace_bytes(b.seqs, heads, b.kv, dim)
    W = be.alloc_bytes(n + (1 << 20))
    be.write_bytes(W, np.full(n + (1 << 20), 0xAB, np.uint8))

    def run():
        be.kv4_attention(Q, b.seqs, b.pool, b.pages, heads, b.kv, dim, scale, Y, W, type=type)
    be.graph_begin()
    run()
    graph = be.graph_end()
    full, starts = b.lengths.copy(), b.starts.copy()
    # rows that lie otherwise, then starts that go back: more tiles than there can be of rows
    apart = np.array([0, 0, *np.arange(1, len(full)) * 3]).astype(np.int32)[:len(full) + 1]
    back = np.where(np.arange(len(full) + 1) % 2, max(r for r, _ in b.sequences), 0).astype(np.int32)
    for keep, at in ((1.0, starts), (0.3, starts), (0.0, starts), (0.7, apart), (1.0, back), (0.5, back), (1.0, starts)):
        be.write(b.seqs.lengths, (full * keep).astype(np.int32))
        be.write(b.seqs.starts, at)
        be.write_bytes(Y, np.zeros(q.size * (2 if type == "bf16" else 4), np.uint8))
        be.graph_launch(graph)
        replayed = be.read_bytes(Y)
        be.write_bytes(Y, np.zeros(q.size * (2 if type == "bf16" else 4), np.uint8))
        run()
        if at is not back:  # sequences that share rows leave either's results
            assert np.array_equal(replayed, be.read_bytes(Y)), keep
        assert np.all(be.read_bytes(W)[n:] == 0xAB)
    be.graph_free(graph)
    got = plain.from_bits(replayed, type)[:q.size].reshape(q.shape).astype(np.float64)
    expect(b, q, got, scale, type, fill=0.0, most=24)
    for buf in (Q, Y, W):
        be.free(buf)
    b.free()
