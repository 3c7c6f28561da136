"""Attention over a 4-bit cache by the kernel of many rows, and by both with
long contexts and in pieces, on the GPU against 64 bits (kv4_plain). test_kv4_rules.py holds
the batches to the kernels. Queries and codes are those whose scores are exact
(test_gpu_kv4): in bf16 a query is one e4m3 number then, and products of eight
neighbours, of one scale, lie less than 2^6 apart. No counterpart in the
reference."""
import numpy as np
import pytest

import kv4_batches as batches
import kv4_plain as plain
from test_gpu_kv4 import LOG2E, Batch, check, gather, limit, queries, reach, run_attention, spread

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(backend):
    yield backend


def batch(be, rng, which, dim, extra_rows=2, **more):
    return Batch(be, rng, which["sequences"], which["kv"], dim, extra_rows=extra_rows, table_pages=which["width"], **more)


def some(b, q, got, scale, type, s, rows, positions=None, window=0, held=None, gate=None):
    """The rows `rows` of sequence s; `held`: its keys and values where not all are numbers."""
    n, length = b.sequences[s]
    k, v = held or b.held(s)
    at = b.starts[s] + np.asarray(rows)
    positions = length - n + np.asarray(rows) if positions is None else positions
    y, size = plain.attention(q[at].astype(np.float64), positions, k, v, scale, window, None if gate is None else gate[at].astype(np.float64))
    exponent = scale * LOG2E * np.abs(q).max() * np.abs(k).sum(-1).max()
    bad = ~(np.abs(got[at] - y) <= limit(size, y, length, exponent, type))
    assert not bad.any(), (s, int(bad.sum()), np.argwhere(bad)[:4], got[at][bad][:4], y[bad][:4])


@pytest.mark.parametrize("type,dim", batches.TYPES)
@pytest.mark.parametrize("name", ["WHOLE", "PIECES"])
def test_attention(be, name, type, dim):
    rng = np.random.default_rng(dim)
    which = getattr(batches, name)
    b = batch(be, rng, which, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    check(b, q, run_attention(be, b, q, scale, type), scale, type)
    b.free()


@pytest.mark.parametrize("type,dim", [t for t in batches.TYPES if t[1] % 64 == 0])
@pytest.mark.parametrize("window", batches.WINDOWS)
def test_window(be, window, type, dim):
    rng = np.random.default_rng(window)
    b = batch(be, rng, batches.WHOLE, dim)
    q = queries(rng, (b.tokens, batches.WHOLE["heads"], dim))
    scale = dim ** -0.5 / 4
    check(b, q, run_attention(be, b, q, scale, type, window=window), scale, type, window=window)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 40), ("bf16", 128), ("bf16", 200), ("f32", 64), ("f32", 104)])
@pytest.mark.parametrize("name,odd", [("WHOLE", False), ("WHOLE", True), ("PIECES", False), ("PIECES", True)])
def test_views_and_gate(be, name, odd, type, dim):
    rng = np.random.default_rng(dim)
    which = getattr(batches, name)
    heads = which["heads"]
    b = batch(be, rng, which, dim)
    q, g = queries(rng, (b.tokens, heads, dim)), plain.bf16(rng.normal(0, 4, (b.tokens, heads, dim)))
    g[0, 0, :4] = [100, -100, 300, -300]
    qv, gv = ((heads * 2 * dim, 2 * dim, 0), (heads * 2 * dim, 2 * dim, dim)) if not odd else ((heads * dim + 11, dim + 1, 3), (heads * dim + 5, dim, 1))
    scale = dim ** -0.5 / 4
    # with 64 heads the odd view's rows overlap: a query is what the memory holds in the end
    q = gather(spread(q, qv, reach(qv, q.shape), np.float32(3)), qv, q.shape)
    got = run_attention(be, b, q, scale, type, gate=g, q_view=qv, gate_view=gv)
    check(b, q, got, scale, type, gate=g)
    b.free()


@pytest.mark.parametrize("type,dim", batches.TYPES)
def test_normal_scores(be, type, dim):
    """Ordinary queries. A score's products are added in f32: 2^-23 of the magnitudes for each of 3 dim additions. In bf16 a query
    is two e4m3 numbers, off by 2^-22 of the row's largest at most, and each of their two products loses up to 7 * 2^-13 of its
    magnitudes where eight neighbours are added, the lower part's being a sixteenth of the higher one's: 7 * 2^-13 (1 + 2^-4)."""
    rng = np.random.default_rng(dim)
    heads = batches.WHOLE["heads"]
    b = batch(be, rng, batches.WHOLE, dim)
    q = rng.normal(0, 1, (b.tokens, heads, dim)).astype(np.float32)
    if type == "bf16":
        q = plain.bf16(q * 2.0 ** rng.integers(-20, 3, q.shape))
    scale = dim ** -0.5
    got = run_attention(be, b, q, scale, type)
    for s, (n, length) in enumerate(b.sequences[:5]):
        k, v = b.held(s)
        a = b.starts[s]
        x = q[a:a + n].astype(np.float64)
        y, size = plain.attention(x, length - n + np.arange(n), k, v, scale)
        per = 3 * dim * 2.0 ** -23 + (7 * 2.0 ** -13 * (1 + 2.0 ** -4) if type == "bf16" else 0)
        products = np.abs(x) @ np.abs(k[:, 0]).max(0)  # of a row, with the largest key of each dimension
        most = scale * LOG2E * products.max()
        lost = scale * (per * products + (2.0 ** -22 * np.abs(x).max(-1) * np.abs(k[:, 0]).sum(-1).max() if type == "bf16" else 0))
        # scores off by e change a probability by exp(e) - 1 and their sum by as much
        off = limit(size, y, length, most, type) + 2 * size * np.expm1(lost)[..., None]
        assert np.all(np.abs(got[a:a + n] - y) <= off)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 128)])
@pytest.mark.parametrize("fill", [0xFF, 0xFE])
def test_what_is_outside_does_not_count(be, fill, type, dim):
    """Positions behind the length, before the window and in pages of others hold NaN or overflow."""
    rng = np.random.default_rng(2)
    window = 65
    b = batch(be, rng, batches.WHOLE, dim)
    held = [b.held(s) for s in range(5)]
    b.host[:] = fill
    for s, (n, length) in enumerate(b.sequences[:5]):
        for p in range(max(0, length - n - window + 1), length):
            plain.put(b.host, b.kv, dim, b.page(s, p), p % 64, held[s][0][p], held[s][1][p])
    b.upload()
    q = queries(rng, (b.tokens, batches.WHOLE["heads"], dim))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type, window=window)
    for s in range(5):
        some(b, q, got, scale, type, s, np.arange(b.sequences[s][0]), window=window, held=held[s])
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 128)])
@pytest.mark.parametrize("at_v,at_k", [(250, 296), (20, 299), (171, 171)])
def test_nan_reaches_the_rows_that_have_it(be, at_v, at_k, type, dim):
    """A block of NaN in a key makes the rows at and behind it NaN, one in a value its 32 dimensions; the other rows stay."""
    rng = np.random.default_rng(3)
    pitch = plain.pitch_of(dim)
    b = batch(be, rng, batches.WHOLE, dim)
    s, (n, length) = 1, b.sequences[1]
    tile = b.host.reshape(-1, 68 * pitch)
    tile[b.page(s, at_k)][64 * pitch + 1 * 64 + at_k % 16 * 4 + at_k % 64 // 16] = 255
    tile[b.page(s, at_v)][66 * pitch + 1 * 64 + at_v // 4 % 4 * 16 + at_v % 64 // 16 * 4 + at_v % 4] = 255
    b.upload()
    q = queries(rng, (b.tokens, batches.WHOLE["heads"], dim))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type)
    a, positions = b.starts[s], length - n + np.arange(n)
    nan = np.zeros((n,) + got.shape[1:], bool)
    nan[positions >= at_v, :, 32:64] = True
    nan[positions >= at_k] = True
    assert np.array_equal(np.isnan(got[a:a + n]), nan)
    k, v = b.held(s)
    y, size = plain.attention(q[a:a + n].astype(np.float64), positions, np.nan_to_num(k), np.nan_to_num(v), scale)
    exponent = scale * LOG2E * 2 * np.nanmax(np.abs(k).sum(-1))
    off = np.abs(got[a:a + n] - y) > limit(size, y, length, exponent, type)
    assert not off[~nan].any()
    assert not np.isnan(np.delete(got, np.arange(a, a + n), 0)).any()
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 128), ("bf16", 256), ("f32", 64)])
def test_queries_that_are_no_numbers(be, type, dim):
    """A query with an infinity or NaN gives its row NaN, and no other."""
    rng = np.random.default_rng(4)
    b = batch(be, rng, batches.WHOLE, dim)
    q = queries(rng, (b.tokens, batches.WHOLE["heads"], dim))
    scale = dim ** -0.5 / 4
    right = run_attention(be, b, q, scale, type)
    wrong = {(3, 5, 1): np.nan, (70, 0, dim - 1): np.inf, (199, 63, 0): -np.inf, (200, 7, 33): np.nan}
    for at, x in wrong.items():
        q[at] = x
    got = run_attention(be, b, q, scale, type)
    for t, h, _ in wrong:
        assert np.all(np.isnan(got[t, h]))
        got[t, h] = right[t, h]
    assert np.array_equal(got, right)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 128)])
def test_pages_that_are_none_and_rows_without_positions(be, type, dim):
    rng = np.random.default_rng(5)
    which = dict(batches.WHOLE, sequences=[(70, 200), (130, 300), (40, 20), (33, 0), (3, 3)] + [(0, 9)] * 19)
    b = batch(be, rng, which, dim)
    b.table[0, [0, 2]] = [-1, b.pages]  # positions 64 to 127 and 192 to 199 are there
    b.table[1, 3:5] = [2 ** 31 - 1, -2 ** 31]  # 0 to 191 are
    be.write(b.seqs.table, b.table)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type)
    both = [plain.get(b.host, 1, dim, b.page(0, p), p % 64) for p in [*range(64, 128), *range(192, 200)]]
    held = tuple(np.stack([x[i] for x in both]) for i in (0, 1))
    position = 130 + np.arange(70)
    some(b, q, got, scale, type, 0, np.arange(70), np.where(position < 192, 63, position - 192 + 64), held=held)
    held = tuple(x[:192] for x in b.held(1, 192))
    some(b, q, got, scale, type, 1, np.arange(130), np.minimum(170 + np.arange(130), 191), held=held)
    a = b.starts[2]
    assert np.all(got[a:a + 20] == 0)
    some(b, q, got, scale, type, 2, np.arange(20, 40), np.arange(20))
    a = b.starts[3]
    assert np.all(got[a:a + 33] == 0)
    some(b, q, got, scale, type, 4, np.arange(3))
    assert np.all(got[b.rows:] == 9)
    be.write(b.seqs.table, np.full_like(b.table, -1))
    assert np.all(run_attention(be, b, q, scale, type)[:b.rows] == 0)
    b.free()


@pytest.mark.parametrize("name", ["WHOLE", "PIECES"])
def test_sequences_that_are_none(be, name):
    """Starts that do not ascend, lengths past the table and more rows than `longest` leave a sequence's rows as they were."""
    rng = np.random.default_rng(6)
    which, dim = getattr(batches, name), 128
    b = batch(be, rng, which, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    right = run_attention(be, b, q, scale, "bf16")
    # a sequence that is none leaves the others' pieces larger or smaller, their sums in another order: two results are each
    # off by 2^-8 of the largest value, 6 * 2^2, and of themselves
    off = 2.0 ** -7 * (24 + np.abs(right))
    for s, length in ((0, 64 * which["width"] + 1), (1, -1), (1, -2 ** 31), (0, 2 ** 31 - 1)):
        lengths = b.lengths.copy()
        lengths[s] = length
        be.write(b.seqs.lengths, lengths)
        got = run_attention(be, b, q, scale, "bf16")
        out = np.arange(b.starts[s], b.starts[s + 1])
        assert np.all(got[out] == 9) and np.all(np.delete(np.abs(got - right) <= off, out, 0))
    be.write(b.seqs.lengths, b.lengths)
    starts = b.starts.copy()
    starts[1] = b.rows + 1  # the first has too many, the second ends before it begins
    be.write(b.seqs.starts, starts)
    got = run_attention(be, b, q, scale, "bf16")
    a = b.starts[2]
    assert np.all(got[:a] == 9) and np.all(np.abs(got[a:] - right[a:]) <= off[a:])
    b.free()


@pytest.mark.parametrize("name,type", [("WHOLE", "bf16"), ("PIECES", "bf16"), ("PIECES", "f32"), ("FEW", "f32"), ("SOME", "bf16")])
def test_captured_and_replayed(be, name, type):
    """A graph takes the lengths and tables that stand there when it runs, as an eager call does."""
    rng = np.random.default_rng(8)
    which, dim, scale = getattr(batches, name), 128, 0.02
    b = batch(be, rng, which, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    size = q.size
    Q, Y = be.alloc(plain.bits(q, type)), be.alloc(plain.bits(np.zeros(size, np.float32), type))
    n = be.kv4_attention_workspace_bytes(b.seqs, which["heads"], b.kv, dim)
    W = be.alloc_bytes(max(4, n))
    be.graph_begin()
    be.kv4_attention(Q, b.seqs, b.pool, b.pages, which["heads"], b.kv, dim, scale, Y, W, type=type)
    graph = be.graph_end()
    full = b.lengths.copy()
    for keep in (1.0, 0.3, 0.0, 0.7, 1.0):
        be.write(b.seqs.lengths, (full * keep).astype(np.int32))
        be.write_bytes(Y, np.zeros(size * (2 if type == "bf16" else 4), np.uint8))
        be.graph_launch(graph)
        replayed = be.read_bytes(Y)
        be.write_bytes(Y, np.zeros(size * (2 if type == "bf16" else 4), np.uint8))
        be.kv4_attention(Q, b.seqs, b.pool, b.pages, which["heads"], b.kv, dim, scale, Y, W, type=type)
        assert np.array_equal(replayed, be.read_bytes(Y))
    be.graph_free(graph)
    got = plain.from_bits(replayed, type)[:size].reshape(q.shape).astype(np.float64)
    for s in (0, 1):
        some(b, q, got, scale, type, s, [0, b.sequences[s][0] - 1])
    for buf in (Q, Y, W):
        be.free(buf)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 64), ("bf16", 192), ("f32", 128)])
@pytest.mark.parametrize("hole", [False, True])
def test_more_than_64_pages(be, hole, type, dim):
    """A workgroup asks for page numbers again every 64 pages."""
    rng = np.random.default_rng(9)
    which = batches.LONG
    b = batch(be, rng, which, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 8
    k, v = b.held(0)
    rows = np.array([0, 63, 64, 100, 129])
    n, length = b.sequences[0]
    positions = length - n + rows
    if hole:
        b.table[0, 65] = -1
        be.write(b.seqs.table, b.table)
        k, v = (np.delete(x, np.arange(65 * 64, 66 * 64), 0) for x in (k, v))
        gone = np.clip(positions - 65 * 64 + 1, 0, 64)
        positions = positions - gone
    some(b, q, run_attention(be, b, q, scale, type), scale, type, 0, rows, positions, held=(k, v))
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 24, 128, 192, 200, 256])
@pytest.mark.parametrize("name", ["FEW", "SOME"])
@pytest.mark.parametrize("window", (0,) + batches.LONG_WINDOWS)
def test_few_rows_in_pieces(be, window, name, dim, type):
    """Sixteen rows a workgroup over a part of the context, with a gate and a page that is none; views that no wide load fits."""
    rng = np.random.default_rng(dim)
    which = getattr(batches, name)
    heads = which["heads"]
    b = batch(be, rng, which, dim)
    q, g = queries(rng, (b.tokens, heads, dim)), plain.bf16(rng.normal(0, 4, (b.tokens, heads, dim)))
    qv, gv = (heads * dim + heads + 11, dim + 1, 3), (heads * dim + 5, dim, 1)
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type, window=window, gate=g, q_view=qv, gate_view=gv)
    check(b, q, got, scale, type, window=window, gate=g)
    if not window:  # positions 64 to 127 of the longest sequence are not there
        b.table[0, 1] = -7
        be.write(b.seqs.table, b.table)
        got = run_attention(be, b, q, scale, type, gate=g, q_view=qv, gate_view=gv)
        n, length = b.sequences[0]
        both = [plain.get(b.host, b.kv, dim, b.page(0, p), p % 64) for p in range(length) if not 64 <= p < 128]
        held = tuple(np.stack([x[i] for x in both]) for i in (0, 1))
        some(b, q, got, scale, type, 0, np.arange(n), length - n - 64 + np.arange(n), held=held, gate=g)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 128), ("f32", 72)])
def test_writing_a_prompt_among_single_tokens(be, type, dim):
    """Rows before position 0, a sequence without positions and one that is none among them; more than 64 sequences."""
    rng = np.random.default_rng(dim)
    sequences = [(1, 100)] * 40 + [(500, 530), (3, 2), (4, 0), (0, 7), (1, 129)] + [(1, 1 + i) for i in range(60)]
    kv = 2
    b = Batch(be, rng, sequences, kv, dim, extra_rows=2, table_pages=9)
    assert (500 + 62) // 64 + 1 > 2 * (b.tokens / 64 / len(sequences) + 2)  # pages of all sequences together
    lengths = b.lengths.copy()
    lengths[-1] = 9 * 64 + 1
    be.write(b.seqs.lengths, lengths)
    k, v = (plain.bf16(rng.normal(0, 1, (b.tokens, kv, dim))) for _ in range(2))
    K, V = (be.alloc(plain.bits(x, type)) for x in (k, v))
    want = b.host.copy()
    back = [np.full(k.shape, 5.0), np.full(k.shape, 5.0)]
    for s, (n, length) in enumerate(sequences[:-1]):
        for i in range(n):
            row, p = b.starts[s] + i, length - n + i
            for x in back:
                x[row] = 0
            if p >= 0:
                plain.put(want, kv, dim, b.page(s, p), p % 64, k[row].astype(np.float64), v[row].astype(np.float64))
                back[0][row], back[1][row] = plain.get(want, kv, dim, b.page(s, p), p % 64)
    be.kv4_write(K, V, b.seqs, b.pool, b.pages, kv, dim, type=type)
    assert np.array_equal(be.read_bytes(b.pool), want)
    for buf in (K, V):
        be.write_bytes(buf, plain.bits(np.full(k.size, 5.0, np.float32), type).view(np.uint8))
    be.kv4_read(b.pool, b.pages, kv, dim, b.seqs, K, V, type=type)
    for buf, x in zip((K, V), back):
        assert np.array_equal(plain.from_bits(be.read_bytes(buf), type)[:k.size].reshape(k.shape), x)
        be.free(buf)
    b.free()


@pytest.mark.parametrize("type,dim", [("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 256)])
def test_a_prompt_among_single_tokens(be, type, dim):
    rng = np.random.default_rng(dim)
    which = batches.MIXED
    b = batch(be, rng, which, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    check(b, q, run_attention(be, b, q, scale, type), scale, type)
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("name,dim", [("LONG_ROWS", 64), ("LONG_ROWS", 192), ("FAR_ROWS", 64)])
def test_long_contexts_of_few_rows(be, name, dim, type):
    """Sixteen rows a workgroup: page numbers asked for again, and more pieces of a row than one turn of the join takes."""
    rng = np.random.default_rng(10)
    which = getattr(batches, name)
    b = batch(be, rng, which, dim)
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 8
    got = run_attention(be, b, q, scale, type)
    for s in (0, 1, len(b.sequences) - 1) if len(b.sequences) > 1 else (0,):
        some(b, q, got, scale, type, s, [0, b.sequences[s][0] - 1])
    b.free()
