"""Attention over a 4-bit key-value cache on the GPU against 64 bits (kv4_plain).

Tolerances are counted from roundings. Queries and what codes stand for are
chosen so that scores are exact in f32 in any order, wherever a case says so
(`exact_scores`): then a probability is off by its exponent's rounding (2^-22 of
the exponent's size, in powers of two) and by the exponential's (2^-22); the
sums of up to `length` positions by 2^-23 each; bf16 adds 2^-8 for the
probability and 2^-8 for the result."""
import numpy as np
import pytest

import kv4_plain as plain

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


@pytest.fixture(scope="module")
def be(backend):
    yield backend


class Batch:
    """Sequences as (rows, length) in a pool, with tables in any order and pages to spare."""

    def __init__(self, be, rng, sequences, kv, dim, extra_rows=0, spare=2, fill="codes", longest=None, table_pages=None):
        import stratacuda_amd as sm
        self.be, self.kv, self.dim, self.sequences = be, kv, dim, sequences
        need = [-(-max(0, n) // 64) for _, n in sequences]
        self.width = table_pages or max(1, max(need))
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(sequences), self.width), -1, np.int32)
        first = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[first:first + n]
            first += n
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
        self.lengths = np.array([n for _, n in sequences], np.int32)
        self.rows = int(self.starts[-1])
        self.tokens = max(1, self.rows + extra_rows)
        nbytes = self.pages * plain.page_bytes(kv, dim)
        if fill == "codes":  # finite numbers everywhere, scales 2^-2 to 2^2
            self.host = rng.integers(0, 256, nbytes, dtype=np.uint8)
            tile = self.host.reshape(-1, 68 * plain.pitch_of(dim))
            tile[:, 64 * plain.pitch_of(dim):] = rng.integers(125, 130, (tile.shape[0], 4 * plain.pitch_of(dim)))
            self.clear_padding()
        else:
            self.host = np.full(nbytes, fill, np.uint8)
        self.pool = be.alloc_bytes(nbytes)
        self.seqs = sm.Sequences(count=len(sequences), tokens=self.tokens,
                                 longest=longest or max(1, max(n for n, _ in sequences)),
                                 starts=be.alloc(self.starts, "i32"), lengths=be.alloc(self.lengths, "i32"),
                                 table=be.alloc(self.table, "i32"), table_pages=self.width)
        self.upload()

    def clear_padding(self):
        """Codes past dim are 0."""
        pitch, dim = plain.pitch_of(self.dim), self.dim
        tile = self.host.reshape(-1, 68 * pitch)
        tile[:, :32 * pitch].reshape(-1, 64, pitch // 2)[:, :, dim // 2:] = 0
        v = tile[:, 32 * pitch:64 * pitch].reshape(-1, pitch // 32, 4, 16, 16)
        for d in range(dim, pitch):
            v[:, d // 32, :, d % 16] &= 0xF0 if d // 16 % 2 == 0 else 0x0F

    def upload(self):
        self.be.write_bytes(self.pool, self.host)

    def page(self, s, at):
        return int(self.table[s, at // 64])

    def held(self, s, length=None):
        """Keys and values [length, kv, dim] of sequence s from the host's copy."""
        length = self.sequences[s][1] if length is None else length
        both = [plain.get(self.host, self.kv, self.dim, self.page(s, p), p % 64) for p in range(length)]
        if not both:
            return np.zeros((0, self.kv, self.dim)), np.zeros((0, self.kv, self.dim))
        return np.stack([k for k, _ in both]), np.stack([v for _, v in both])

    def free(self):
        for b in (self.pool, self.seqs.starts, self.seqs.lengths, self.seqs.table):
            self.be.free(b)


def spread(x, view, size, fill):
    """x [t, h, d] laid out by the view in an array of `size` values filled with `fill`."""
    out = np.full(size, fill, x.dtype)
    t, h, d = np.indices(x.shape)
    out[t * view[0] + h * view[1] + view[2] + d] = x
    return out


def gather(flat, view, shape):
    t, h, d = np.indices(shape)
    return flat[t * view[0] + h * view[1] + view[2] + d]


def reach(view, shape):
    return (shape[0] - 1) * view[0] + (shape[1] - 1) * view[1] + view[2] + shape[2]


# ------------------------------------------------------------- write and read
VALUES = {
    "normal": lambda rng, shape: rng.normal(0, 1, shape),
    "far": lambda rng, shape: rng.normal(0, 1, shape) * 10.0 ** rng.uniform(-30, 30, shape),
    # multiples of a quarter step around each code: every tie
    "ties": lambda rng, shape: rng.integers(-24, 25, shape) * 0.25,
    "zeros": lambda rng, shape: np.where(rng.random(shape) < 0.9, 0.0, rng.choice([-0.0, 6.0, 2.0 ** -126, -(2.0 ** -128), 3e38], shape)),
    "odd": lambda rng, shape: np.where(rng.random(shape) < 0.01, rng.choice([np.inf, -np.inf, np.nan], shape), rng.normal(0, 1, shape)),
    "edges": lambda rng, shape: rng.choice([6.0, 6.0000005, 5.9999995, 3.4028235e38, 2.0 ** 127, 1e-45, 2.0 ** -124, 0.0], shape),
}


def typed(x, type):
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore"):
        return x.astype(np.float32) if type == "f32" else bf16_any(x)


def bf16_any(x):
    """f32 values that bf16 holds: x cut to 8 significant bits."""
    u = x.astype(np.float32).view(np.uint32) & 0xffff0000
    return u.view(np.float32)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("dim,kv,views", [(128, 2, 0), (256, 1, 0), (64, 3, 1), (80, 2, 2), (8, 1, 0), (40, 5, 1), (96, 1, 2), (192, 2, 0), (200, 1, 1)])
def test_write_and_read(be, dim, kv, views, type):
    """Bytes written in steps of all sizes are those of the definition, no other byte changes, and they read back as its numbers."""
    rng = np.random.default_rng(dim + kv)
    for kind, steps in zip(VALUES, ([1, 1, 62, 1, 5], [70], [3, 61, 64], [130, 1], [64, 1, 63], [2, 3])):
        b = Batch(be, rng, [(0, sum(steps)), (0, 1), (0, 70)], kv, dim)
        before = b.host.copy()
        done = 0
        for n in steps:
            rows = [n, 0, n % 71]
            lengths = [done + n, 1, max(70 - done, rows[2])][:3]
            lengths[2] = min(70, max(lengths[2], rows[2]))
            rows[2] = min(rows[2], lengths[2])
            tokens = sum(rows) + 1
            k, v = (typed(VALUES[kind](rng, (tokens, kv, dim)), type) for _ in range(2))
            kview = [(kv * dim, dim, 0), (2 * kv * dim + 8, 2 * dim, 16), (kv * dim + 3, dim + 1, 5)][views]
            vview = [(kv * dim, dim, 0), (2 * kv * dim + 8, 2 * dim, 16 + dim), (kv * dim + 3, dim + 1, 2)][views]
            size = max(reach(kview, k.shape), reach(vview, v.shape))
            K, V = (be.alloc(plain.bits(spread(x, w, size, np.float32(7)), type)) for x, w in ((k, kview), (v, vview)))
            starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
            be.write(b.seqs.starts, starts)
            be.write(b.seqs.lengths, np.array(lengths, np.int32))
            seqs = b.seqs._replace(tokens=tokens, longest=max(rows))
            be.kv4_write(K, V, seqs, b.pool, b.pages, kv, dim, k_view=kview, v_view=vview, type=type)
            for s in range(3):
                for i in range(rows[s]):
                    p = lengths[s] - rows[s] + i
                    plain.put(before, kv, dim, b.page(s, p), p % 64, k[starts[s] + i].astype(np.float64), v[starts[s] + i].astype(np.float64))
            got = be.read_bytes(b.pool)
            assert np.array_equal(got, before), (kind, n, np.flatnonzero(got != before)[:8])
            # and back, into views with other things between the rows
            out = [be.alloc(plain.bits(np.full(size, 7, np.float32), type)) for _ in range(2)]
            be.kv4_read(b.pool, b.pages, kv, dim, seqs, out[0], out[1], k_view=kview, v_view=vview, type=type)
            b.host = got
            for buf, view, which in ((out[0], kview, 0), (out[1], vview, 1)):
                want = np.full(size, 7, np.float64)
                for s in range(3):
                    for i in range(rows[s]):
                        p = lengths[s] - rows[s] + i
                        x = plain.get(got, kv, dim, b.page(s, p), p % 64)[which]
                        t, h, d = np.indices((1, kv, dim))
                        want[((starts[s] + i) * view[0] + h * view[1] + view[2] + d)[0]] = x
                raw = plain.from_bits(be.read_bytes(buf), type)[:size]
                assert np.array_equal(raw.astype(np.float64), want, equal_nan=True), (kind, n)
            for buf in [K, V] + out:
                be.free(buf)
            done += n
        b.free()


def test_read_of_no_page(be):
    """Positions whose page number is outside the pool read as 0, and are not written."""
    rng = np.random.default_rng(1)
    kv, dim = 2, 64
    b = Batch(be, rng, [(200, 200), (5, 3)], kv, dim)
    b.table[0, 1] = b.pages
    b.table[0, 2] = -7
    be.write(b.seqs.table, b.table)
    K, V = (be.alloc(np.full(205 * kv * dim, 3, np.float32)) for _ in range(2))
    be.kv4_read(b.pool, b.pages, kv, dim, b.seqs, K, V)
    for buf, which in ((K, 0), (V, 1)):
        got = be.read(buf).reshape(205, kv, dim)
        for p in range(200):
            want = 0 if 64 <= p < 192 else plain.get(b.host, kv, dim, b.page(0, p), p % 64)[which]
            assert np.array_equal(got[p], np.broadcast_to(want, (kv, dim)))
        for i in range(5):  # two rows before position 0
            want = 0 if i < 2 else plain.get(b.host, kv, dim, b.page(1, 0), i - 2)[which]
            assert np.array_equal(got[200 + i], np.broadcast_to(want, (kv, dim)))
    want = b.host.copy()
    x = np.arange(205 * kv * dim, dtype=np.float32).reshape(205, kv, dim) % 7
    be.write(K, x)
    be.write(V, -x)
    be.kv4_write(K, V, b.seqs, b.pool, b.pages, kv, dim)
    for p in range(200):
        if not 64 <= p < 192:
            plain.put(want, kv, dim, b.page(0, p), p % 64, x[p], -x[p])
    for i in range(2, 5):
        plain.put(want, kv, dim, b.page(1, 0), i - 2, x[200 + i], -x[200 + i])
    assert np.array_equal(be.read_bytes(b.pool), want)
    b.free()


# ------------------------------------------------------------------ attention
def queries(rng, shape):
    return rng.choice([0, 0.5, -0.5, 1, -1, 2, -2], shape).astype(np.float32)


def limit(size, y, length, exponent, type):
    """How far a result may be off: `size` is the sum of p |v| over l, `exponent` the largest exponent in powers of two."""
    off = size * (2.0 ** -21 * (2 + exponent) + (length + 64) * 2.0 ** -22)
    return off + (2.0 ** -8 * size + 2.0 ** -8 * np.abs(y) if type == "bf16" else 0) + 1e-30


def run_attention(be, b, q, scale, type, window=0, gate=None, q_view=None, gate_view=None, fill=9.0, heads=None):
    heads = q.shape[1]
    dim = b.dim
    qv = q_view or (heads * dim, dim, 0)
    Q = be.alloc(plain.bits(spread(q, qv, reach(qv, q.shape), np.float32(3)), type))
    G = None
    if gate is not None:
        gv = gate_view or (heads * dim, dim, 0)
        G = be.alloc(plain.bits(spread(gate, gv, reach(gv, gate.shape), np.float32(3)), type))
    Y = be.alloc(plain.bits(np.full(b.tokens * heads * dim, fill, np.float32), type))
    n = be.kv4_attention_workspace_bytes(b.seqs, heads, b.kv, dim)
    W = be.alloc_bytes(n) if n else None
    if W:
        be.write_bytes(W, np.full(n, 0xFF, np.uint8))  # nothing in it matters
    be.kv4_attention(Q, b.seqs, b.pool, b.pages, heads, b.kv, dim, scale, Y, W, window=window, gate=G, q_view=q_view,
                     gate_view=gate_view, type=type)
    got = plain.from_bits(be.read_bytes(Y), type)[:b.tokens * heads * dim].reshape(b.tokens, heads, dim).astype(np.float64)
    for buf in (Q, G, Y, W):
        if buf:
            be.free(buf)
    return got


def check(b, q, got, scale, type, window=0, gate=None, fill=9.0):
    for s, (n, length) in enumerate(b.sequences):
        k, v = b.held(s)
        a = b.starts[s]
        y, size = plain.attention(q[a:a + n].astype(np.float64), length - n + np.arange(n), k, v, scale, window,
                                  None if gate is None else gate[a:a + n].astype(np.float64))
        exponent = scale * LOG2E * np.abs(q).max() * (np.abs(k).sum(-1).max() if k.size else 0)
        bad = np.abs(got[a:a + n] - y) > limit(size, y, length, exponent, type)
        assert not bad.any(), (s, int(bad.sum()), np.argwhere(bad)[:4], got[a:a + n][bad][:4], y[bad][:4])
    assert np.all(got[b.rows:] == fill)


SHAPES = [(24, 2, 256), (32, 8, 128), (8, 8, 64), (4, 1, 128), (40, 2, 64), (12, 4, 80), (6, 2, 192), (5, 5, 40), (2, 1, 8), (34, 2, 96), (3, 1, 200)]
BATCHES = {
    "one": [(1, 1)],
    "token": [(1, 300)],
    "page": [(1, 64), (1, 65), (1, 63), (1, 128)],
    "few": [(3, 90), (1, 5), (8, 8), (2, 200)],
    "prompts": [(70, 70), (33, 170), (0, 40), (1, 129), (130, 131)],
}


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_attention(be, heads, kv, dim, name, type):
    rng = np.random.default_rng(heads * dim)
    b = Batch(be, rng, BATCHES[name], kv, dim, extra_rows=3)
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 4
    check(b, q, run_attention(be, b, q, scale, type), scale, type)
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100])
@pytest.mark.parametrize("heads,kv,dim", [(24, 2, 256), (8, 4, 64), (4, 1, 128)])
def test_window(be, heads, kv, dim, window, type):
    rng = np.random.default_rng(window)
    b = Batch(be, rng, [(1, 200), (100, 150), (66, 66), (1, 1)], kv, dim)
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 4
    check(b, q, run_attention(be, b, q, scale, type, window=window), scale, type, window=window)
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,odd", [(1, False), (40, False), (1, True), (150, True)])
def test_views_and_gate(be, rows, odd, type):
    """Queries beside their gates as a projection leaves them, and views that no load of 16 bytes fits."""
    rng = np.random.default_rng(rows)
    heads, kv, dim = 6, 2, 128
    b = Batch(be, rng, [(rows, 170), (1, 3)], kv, dim)
    q, g = queries(rng, (b.tokens, heads, dim)), plain.bf16(rng.normal(0, 4, (b.tokens, heads, dim)))
    g[0, 0, :4] = [100, -100, 300, -300]
    qv, gv = ((heads * 2 * dim, 2 * dim, 0), (heads * 2 * dim, 2 * dim, dim)) if not odd else ((heads * dim + 11, dim + 1, 3), (heads * dim + 5, dim, 1))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type, gate=g, q_view=qv, gate_view=gv)
    check(b, q, got, scale, type, gate=g)
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(24, 2, 256), (4, 2, 80)])
def test_normal_scores(be, heads, kv, dim, type):
    """Ordinary queries, whose scores are rounded: 2^-23 for each of a score's 3 dim additions (2^-8 of nothing: bf16 queries are
    taken as they are), on top of the rest."""
    rng = np.random.default_rng(5)
    b = Batch(be, rng, [(1, 400), (20, 90)], kv, dim)
    q = rng.normal(0, 1, (b.tokens, heads, dim)).astype(np.float32)
    if type == "bf16":
        q = plain.bf16(q)
    scale = dim ** -0.5
    got = run_attention(be, b, q, scale, type)
    for s, (n, length) in enumerate(b.sequences):
        k, v = b.held(s)
        a = b.starts[s]
        y, size = plain.attention(q[a:a + n].astype(np.float64), length - n + np.arange(n), k, v, scale)
        most = scale * LOG2E * (np.abs(q).max(0).max(0) * np.abs(k).max((0, 1))).sum()
        off = limit(size, y, length, most, type) + 2 * size * most * 3 * dim * 2.0 ** -23
        assert np.all(np.abs(got[a:a + n] - y) <= off)
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("fill", [0xFF, 0xFE])
def test_what_is_outside_does_not_count(be, fill, type):
    """Positions behind the length, before the window and in pages of others hold NaN or overflow."""
    rng = np.random.default_rng(2)
    heads, kv, dim, window = 12, 2, 128, 70
    b = Batch(be, rng, [(1, 130), (20, 140), (1, 1)], kv, dim)
    held = [b.held(s) for s in range(3)]
    b.host[:] = fill
    for s, (n, length) in enumerate(b.sequences):
        for p in range(max(0, length - n - window + 1), length):
            plain.put(b.host, kv, dim, b.page(s, p), p % 64, held[s][0][p], held[s][1][p])
    b.upload()
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type, window=window)
    for s, (n, length) in enumerate(b.sequences):
        a = b.starts[s]
        y, size = plain.attention(q[a:a + n].astype(np.float64), length - n + np.arange(n), held[s][0], held[s][1], scale, window)
        exponent = scale * LOG2E * 2 * np.abs(held[s][0]).sum(-1).max()
        assert np.all(np.abs(got[a:a + n] - y) <= limit(size, y, length, exponent, type))
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [30, 150])
def test_nan_reaches_the_rows_that_have_it(be, rows, type):
    """A block of NaN in a key makes the rows at and behind it NaN, one in a value its 32 dimensions; the rows before stay."""
    rng = np.random.default_rng(3)
    heads, kv, dim = 6, 2, 128
    b = Batch(be, rng, [(rows, rows + 10)], kv, dim)
    at_v, at_k = rows // 2, rows - 4
    for p, part in ((at_v, 66), (at_k, 64)):
        pitch, r = 128, p % 64
        tile = b.host.reshape(-1, 68 * pitch)[b.page(0, p) * kv + 1]
        if part == 64:
            tile[64 * pitch + 2 * 64 + r % 16 * 4 + r // 16] = 255
        else:
            tile[66 * pitch + 1 * 64 + r // 4 % 4 * 16 + r // 16 * 4 + r % 4] = 255
    b.upload()
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type)
    k, v = b.held(0)
    positions = 10 + np.arange(rows)
    nan = np.zeros(got.shape, bool)
    nan[np.ix_(positions >= at_v, [3, 4, 5], range(32, 64))] = True
    nan[np.ix_(positions >= at_k, [3, 4, 5])] = True
    assert np.array_equal(np.isnan(got), nan)
    y, size = plain.attention(q.astype(np.float64), positions, np.nan_to_num(k), np.nan_to_num(v), scale)
    exponent = scale * LOG2E * 2 * np.nanmax(np.abs(k).sum(-1))
    off = np.abs(got - y) > limit(size, y, rows + 10, exponent, type)
    assert not off[~nan].any()
    b.free()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 100])
def test_rows_without_positions(be, rows, type):
    """Rows before position 0, sequences of length 0 and pages that are none give 0."""
    rng = np.random.default_rng(4)
    heads, kv, dim = 4, 2, 64
    b = Batch(be, rng, [(rows, 0), (rows + 2, rows), (rows, 256)], kv, dim, extra_rows=2)
    b.table[2, :3] = [-1, b.pages, 2 ** 31 - 1]  # 192 of 256 positions are not there
    be.write(b.seqs.table, b.table)
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 4
    got = run_attention(be, b, q, scale, type)
    assert np.all(got[:rows + 2] == 0)
    k, v = b.held(1)
    a = b.starts[1]
    y, size = plain.attention(q[a:a + rows + 2].astype(np.float64), np.arange(-2, rows), k, v, scale)
    assert np.all(np.abs(got[a:a + rows + 2] - y) <= limit(size, y, 256, 100, type))
    a = b.starts[2]
    both = [plain.get(b.host, kv, dim, b.page(2, p), p % 64) for p in range(192, 256)]
    k, v = (np.stack([x[i] for x in both]) for i in (0, 1))
    y, size = plain.attention(q[a:a + rows].astype(np.float64), 256 - rows + np.arange(rows) - 192, k, v, scale)
    assert np.all(np.abs(got[a:a + rows] - y) <= limit(size, y, 256, 100, type))
    assert np.all(got[b.rows:] == 9)
    # no page at all
    be.write(b.seqs.table, np.full_like(b.table, -1))
    assert np.all(run_attention(be, b, q, scale, type)[:b.rows] == 0)
    b.free()


@pytest.mark.parametrize("rows", [1, 90])
def test_sequences_that_are_none(be, rows):
    """Starts that do not ascend or leave the rows, lengths past the table and more rows than `longest` leave a sequence out; the
    others are computed."""
    rng = np.random.default_rng(6)
    heads, kv, dim = 4, 2, 64
    b = Batch(be, rng, [(rows, 100)] * 5, kv, dim, table_pages=2)
    q = queries(rng, (b.tokens, heads, dim))
    scale = dim ** -0.5 / 4
    right = run_attention(be, b, q, scale, "f32")
    n = rows
    for starts, lengths, kept in (([0, n, 2 * n, 3 * n, 4 * n, 5 * n], [100, 129, -1, 2 ** 31 - 1, 100], [0, 4]),
                                  ([0, n, n - 1, 3 * n, 4 * n, 5 * n + 1], [100] * 5, [0, 3]),
                                  ([-1, n, 2 * n, 3 * n, 4 * n, -2 ** 31], [100] * 5, [1, 2, 3])):
        be.write(b.seqs.starts, np.array(starts, np.int32))
        be.write(b.seqs.lengths, np.array(lengths, np.int32))
        got = run_attention(be, b, q, scale, "f32")
        for s in range(5):
            want = right[s * n:(s + 1) * n] if s in kept else np.full_like(right[:n], 9)
            if starts[s:s + 2] == [n - 1, 3 * n]:  # rows it shares with none, if they are not too many
                continue
            assert np.array_equal(got[s * n:(s + 1) * n], want), (starts, s)
        before = be.read_bytes(b.pool)
        x = be.alloc(np.ones(b.tokens * kv * dim, np.float32))
        be.kv4_write(x, x, b.seqs, b.pool, b.pages, kv, dim)
        after = be.read_bytes(b.pool).reshape(b.pages, -1)
        changed = set(np.flatnonzero((after != before.reshape(b.pages, -1)).any(1)))
        for s in range(5):
            if s not in kept and starts[s:s + 2] != [n - 1, 3 * n]:
                assert not changed & set(b.table[s].tolist()), (starts, s)
        be.write_bytes(b.pool, before)
        be.free(x)
    b.free()


def test_large_scores_and_one_position_far_above(be):
    """One position whose score is far above the others, late in the context, and scores of a thousand powers of two."""
    rng = np.random.default_rng(7)
    heads, kv, dim = 16, 1, 128
    b = Batch(be, rng, [(1, 1000)], kv, dim)
    k, v = b.held(0)
    peak = 700
    k[peak] = 6 * np.sign(rng.normal(0, 1, (kv, dim)))
    plain.put(b.host, kv, dim, b.page(0, peak), peak % 64, k[peak], v[peak])
    b.upload()
    q = np.broadcast_to(np.sign(k[peak]) * 2, (1, heads, dim)).astype(np.float32).copy()
    for scale in (1.0, 0.01):
        got = run_attention(be, b, q, scale, "f32")
        y, size = plain.attention(q.astype(np.float64), [999], k, v, scale)
        assert np.all(np.abs(got - y) <= limit(size, y, 1000, scale * LOG2E * 1536, "f32"))
    b.free()


@pytest.mark.parametrize("rows", [1, 70])
def test_captured_and_replayed(be, rows):
    """A graph of the write and the attention takes the lengths and tables that stand there when it runs."""
    rng = np.random.default_rng(8)
    heads, kv, dim, scale = 8, 2, 128, 0.02
    b = Batch(be, rng, [(rows, 300), (1, 200)], kv, dim)
    q = queries(rng, (b.tokens, heads, dim))
    Q, Y = be.alloc(q), be.alloc(np.zeros(q.size, np.float32))
    x = rng.normal(0, 1, (b.tokens, kv, dim)).astype(np.float32)
    X = be.alloc(x)
    W = be.alloc_bytes(max(4, be.kv4_attention_workspace_bytes(b.seqs, heads, kv, dim)))
    be.graph_begin()
    be.kv4_write(X, X, b.seqs, b.pool, b.pages, kv, dim)
    be.kv4_attention(Q, b.seqs, b.pool, b.pages, heads, kv, dim, scale, Y, W)
    graph = be.graph_end()
    for lengths in ([300, 200], [rows, 1], [100, 77], [257, 200]):
        be.write(b.seqs.lengths, np.array(lengths, np.int32))
        be.graph_launch(graph)
        replayed, pool = be.read(Y), be.read_bytes(b.pool)
        be.kv4_write(X, X, b.seqs, b.pool, b.pages, kv, dim)
        be.kv4_attention(Q, b.seqs, b.pool, b.pages, heads, kv, dim, scale, Y, W)
        assert np.array_equal(replayed, be.read(Y)) and np.array_equal(pool, be.read_bytes(b.pool))
        b.host, b.sequences = pool, [(rows, lengths[0]), (1, lengths[1])]
        check(b, q, replayed.reshape(q.shape).astype(np.float64), scale, "f32")
    be.graph_free(graph)
    for buf in (Q, Y, X, W):
        be.free(buf)
    b.free()


def test_offsets_past_32_bits(be):
    """Pages on both sides of 2^32 bytes in a pool."""
    rng = np.random.default_rng(9)
    import stratacuda_amd as sm
    kv, dim, heads = 8, 256, 16
    each = plain.page_bytes(kv, dim)
    pages = 2 ** 32 // each + 40
    pool = be.alloc_bytes(pages * each)
    table = np.array([[2 ** 32 // each + 1, 5, pages - 1], [2 ** 32 // each, 2 ** 31 // each, 0]], np.int32)
    lengths = [150, 130]
    n = sum(lengths)
    seqs = sm.Sequences(count=2, tokens=n, longest=150, starts=be.alloc(np.array([0, 150, 280], np.int32)),
                        lengths=be.alloc(np.array(lengths, np.int32)), table=be.alloc(table), table_pages=3)
    k, v = (plain.bf16(rng.normal(0, 1, (n, kv, dim))) for _ in range(2))
    K, V = be.alloc(k), be.alloc(v)
    be.kv4_write(K, V, seqs, pool, pages, kv, dim)
    k, v = (plain.numbers(*plain.quantize(x.astype(np.float64))) for x in (k, v))
    be.kv4_read(pool, pages, kv, dim, seqs, K, V)
    assert np.array_equal(be.read(K).reshape(k.shape), k) and np.array_equal(be.read(V).reshape(v.shape), v)
    q = queries(rng, (n, heads, dim))
    Q, Y = be.alloc(q), be.alloc(np.zeros(q.size, np.float32))
    W = be.alloc_bytes(max(4, be.kv4_attention_workspace_bytes(seqs, heads, kv, dim)))
    be.kv4_attention(Q, seqs, pool, pages, heads, kv, dim, 0.02, Y, W)
    got = be.read(Y).reshape(q.shape)
    for a, length in ((0, 150), (150, 130)):
        pos = np.array([0, 63, 64, length - 1])
        y, size = plain.attention(q[a + pos].astype(np.float64), pos, k[a:a + length], v[a:a + length], 0.02)
        # scores are sums of 3 * 256 rounded numbers here
        assert np.all(np.abs(got[a + pos] - y) <= limit(size, y, length, 40, "f32") + 2 * size * 40 * 768 * 2.0 ** -23)
    for buf in (pool, K, V, Q, Y, W, seqs.starts, seqs.lengths, seqs.table):
        be.free(buf)


def test_more_sequences_than_a_wave(be):
    rng = np.random.default_rng(10)
    heads, kv, dim = 4, 2, 64
    for sequences in ([(1, 1 + 7 * i % 150) for i in range(150)], [(i % 3, 70 * (i % 5) + 3) for i in range(70)]):
        b = Batch(be, rng, sequences, kv, dim, extra_rows=1)
        q = queries(rng, (b.tokens, heads, dim))
        check(b, q, run_attention(be, b, q, 0.03, "f32"), 0.03, "f32")
        b.free()


# ------------------------------------------------------------ norm and rotate
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("dim,rotary,heads,kv", [(256, 64, 24, 2), (128, 128, 8, 8), (64, 32, 5, 1), (80, 80, 4, 2), (96, 24, 3, 3), (8, 2, 1, 1),
                                                 (40, 10, 2, 1), (16, 16, 2, 2), (200, 180, 2, 1), (24, 14, 1, 1), (256, 256, 1, 1)])
def test_norm_rope(be, dim, rotary, heads, kv, type):
    """n is off by 4 roundings of f32 (its factor, gamma, two products), a turned one by two products and a sum more: 2^-21 of the
    two terms' sizes covers them; bf16 adds its rounding."""
    rng = np.random.default_rng(dim + rotary)
    context = 300
    cos, sin = (f(rng.uniform(0, 7, (context, rotary // 2))).astype(np.float32) for f in (np.cos, np.sin))
    for tokens, odd in ((1, False), (33, False), (7, True)):
        positions = rng.integers(0, context, tokens).astype(np.int32)
        positions[0] = context - 1
        qv = (2 * heads * dim, 2 * dim, dim) if not odd else (heads * dim + 7, dim + 1, 3)
        kview = (kv * dim + 16, dim, 8) if not odd else None
        x = {n: typed(rng.normal(0, 1, (tokens, h, dim)) * 10.0 ** rng.integers(-3, 4, (tokens, h, 1)), type) for n, h in (("q", heads), ("k", kv))}
        gamma = {n: rng.normal(1, 0.2, dim).astype(np.float32) for n in x}
        flat = {n: spread(x[n], w, reach(w, x[n].shape) + 1, np.float32(5)) for n, w in (("q", qv), ("k", kview or (kv * dim, dim, 0)))}
        x["q"] = gather(flat["q"], qv, x["q"].shape)  # the odd view's rows overlap: what lies there in the end
        bufs = dict(q=be.alloc(plain.bits(flat["q"], type)), k=be.alloc(plain.bits(flat["k"], type)),
                    qg=be.alloc(gamma["q"]), kg=be.alloc(gamma["k"]), cos=be.alloc(cos), sin=be.alloc(sin), at=be.alloc(positions, "i32"),
                    yq=be.alloc(plain.bits(np.zeros(x["q"].size, np.float32), type)), yk=be.alloc(plain.bits(np.zeros(x["k"].size, np.float32), type)))
        be.qk_norm_rope(bufs["q"], bufs["k"], tokens, heads, kv, dim, bufs["qg"], bufs["kg"], 1e-6, bufs["cos"], bufs["sin"], rotary, context,
                        bufs["at"], bufs["yq"], bufs["yk"], q_view=qv, k_view=kview, type=type)
        for n, out in (("q", "yq"), ("k", "yk")):
            got = plain.from_bits(be.read_bytes(bufs[out]), type).reshape(x[n].shape).astype(np.float64)
            y, normed = plain.norm_rope(x[n], gamma[n], np.float32(1e-6).astype(np.float64), cos, sin, rotary, positions)
            half = rotary // 2
            size = np.abs(normed)
            size[..., :rotary] = np.tile(np.abs(normed[..., :half]) + np.abs(normed[..., half:rotary]), 2)
            off = size * 2.0 ** -21 + (np.abs(y) * 2.0 ** -8 if type == "bf16" else 0)
            bad = np.abs(got - y) > off
            assert not bad.any(), (tokens, n, int(bad.sum()))
        for buf in bufs.values():
            be.free(buf)


def test_norm_rope_range(be):
    """Rows of large values, of subnormal ones with eps 0, and positions outside the tables."""
    dim, rotary, context = 64, 32, 4
    cos, sin = np.full((context, 16), 0.6, np.float32), np.full((context, 16), 0.8, np.float32)
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (5, 1, dim)).astype(np.float64)
    x[0] *= 1e38 / np.abs(x[0]).max()
    x[1] *= 1e-40
    x = x.astype(np.float32)
    positions = np.array([0, 3, -1, 4, 2 ** 31 - 1], np.int32)
    q, ones, c, s, at = be.alloc(x), be.alloc(np.ones(dim, np.float32)), be.alloc(cos), be.alloc(sin), be.alloc(positions, "i32")
    yq, yk = be.alloc(np.zeros(x.size, np.float32)), be.alloc(np.zeros(x.size, np.float32))
    be.qk_norm_rope(q, q, 5, 1, 1, dim, ones, ones, 0.0, c, s, rotary, context, at, yq, yk)
    got = be.read(yq).reshape(x.shape).astype(np.float64)
    assert np.array_equal(be.read(yk).reshape(x.shape), got, equal_nan=True)
    y, normed = plain.norm_rope(x, np.ones(dim), 0.0, cos, sin, rotary, np.zeros(5, int))
    assert np.all(np.abs(got[:2] - y[:2]) <= 2.0 ** -20 * np.abs(normed[:2]).max())
    assert np.isnan(got[2:, :, :rotary]).all()
    assert np.all(np.abs(got[2:, :, rotary:] - normed[2:, :, rotary:]) <= 2.0 ** -21 * np.abs(normed[2:, :, rotary:]))
    for buf in (q, ones, c, s, at, yq, yk):
        be.free(buf)


# ------------------------------------------------------------------- together
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_a_layer_step_by_step(be, type):
    """Norm and rotation, write, attention with its gate, a prompt and then tokens: as the plain operators give it from the same
    rounded queries, and the pool's own numbers."""
    import stratacuda_amd as sm
    rng = np.random.default_rng(11)
    heads, kv, dim, rotary, context, scale = 12, 2, 128, 64, 400, 128 ** -0.5
    angles = np.arange(context)[:, None] * 10000.0 ** (-np.arange(rotary // 2) * 2 / rotary)
    cos, sin = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    gammas = [rng.normal(1, 0.1, dim).astype(np.float32) for _ in range(2)]
    qg, kg, c, s = (be.alloc(x) for x in (*gammas, cos, sin))
    table = np.array([[3, 0, 5, 1], [4, 2, 7, 6]], np.int32)
    pool = be.alloc_bytes(be.kv4_bytes(8, kv, dim))
    bufs = [qg, kg, c, s, pool]
    lengths = np.zeros(2, int)
    for new in ([100, 37], [1, 1], [1, 0], [5, 64], [1, 1]):
        lengths += new
        n = sum(new)
        starts = np.concatenate([[0], np.cumsum(new)])
        positions = np.concatenate([lengths[i] - new[i] + np.arange(new[i]) for i in range(2)])
        full, k, v = (typed(rng.normal(0, 1, shape), type) for shape in ((n, heads, 2 * dim), (n, kv, dim), (n, kv, dim)))
        F, K, V = (be.alloc(plain.bits(x, type)) for x in (full, k, v))
        Yq, Yk, Y = (be.alloc(plain.bits(np.zeros(n * h * dim, np.float32), type)) for h in (heads, kv, heads))
        seqs = sm.Sequences(count=2, tokens=n, longest=max(new), starts=be.alloc(starts.astype(np.int32)),
                            lengths=be.alloc(lengths.astype(np.int32)), table=be.alloc(table), table_pages=4)
        at = be.alloc(positions.astype(np.int32))
        qv, gv = (heads * 2 * dim, 2 * dim, 0), (heads * 2 * dim, 2 * dim, dim)
        be.qk_norm_rope(F, K, n, heads, kv, dim, qg, kg, 1e-6, c, s, rotary, context, at, Yq, Yk, q_view=qv, type=type)
        be.kv4_write(Yk, V, seqs, pool, 8, kv, dim, type=type)
        W = be.alloc_bytes(max(4, be.kv4_attention_workspace_bytes(seqs, heads, kv, dim)))
        be.kv4_attention(Yq, seqs, pool, 8, heads, kv, dim, scale, Y, W, gate=F, gate_view=gv, type=type)
        q = plain.from_bits(be.read_bytes(Yq), type)[:n * heads * dim].reshape(n, heads, dim)
        yk = plain.from_bits(be.read_bytes(Yk), type)[:n * kv * dim].reshape(n, kv, dim)
        got = plain.from_bits(be.read_bytes(Y), type)[:n * heads * dim].reshape(n, heads, dim)
        host = be.read_bytes(pool)
        for i in range(2):
            if not new[i]:
                continue
            both = [plain.get(host, kv, dim, table[i, p // 64], p % 64) for p in range(lengths[i])]
            kk, vv = (np.stack([x[j] for x in both]) for j in (0, 1))
            rows = slice(starts[i], starts[i + 1])
            assert np.array_equal(kk[lengths[i] - new[i]:], plain.numbers(*plain.quantize(yk[rows].astype(np.float64))))
            assert np.array_equal(vv[lengths[i] - new[i]:], plain.numbers(*plain.quantize(v[rows].astype(np.float64))))
            y, size = plain.attention(q[rows].astype(np.float64), positions[rows], kk, vv, scale, gate=full[rows, :, dim:].astype(np.float64))
            most = scale * LOG2E * (np.abs(q).max((0, 1)) * np.abs(kk).max((0, 1))).sum()
            off = limit(size, y, lengths[i], most, type) + 2 * size * most * 3 * dim * 2.0 ** -23
            assert np.all(np.abs(got[rows] - y) <= off)
        for buf in (F, K, V, Yq, Yk, Y, at, W, seqs.starts, seqs.lengths, seqs.table):
            be.free(buf)
    for buf in bufs:
        be.free(buf)
