"""Sequences that are none, beside others whose results stay exact: where no
sequence is cut they keep every bit, in pieces (whose sizes go by all
sequences' pages) they are those of 64 bits. No counterpart in the reference."""
import numpy as np
import pytest

import kv4_batches as batches
from kv4_compare import expect
from test_gpu_kv4 import Batch, queries, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(backend):
    yield backend


@pytest.mark.parametrize("type,dim", [("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("name,whole", [("WHOLE", True), ("PIECES", False), ("FEW", False), ("SOME", False), ("MIXED", True)])
def test_the_others_are_computed(be, name, whole, type, dim):
    rng = np.random.default_rng(6)
    which = getattr(batches, name)
    b = Batch(be, rng, which["sequences"], which["kv"], dim, extra_rows=2, table_pages=which["width"])
    q = queries(rng, (b.tokens, which["heads"], dim))
    scale = dim ** -0.5 / 4
    right = run_attention(be, b, q, scale, type)
    expect(b, q, right, scale, type)

    def others(left):
        got = run_attention(be, b, q, scale, type)
        expect(b, q, got, scale, type, left=left)
        if whole:
            for s in range(len(b.sequences)):
                rows = slice(b.starts[s], b.starts[s + 1])
                assert s in left or np.array_equal(got[rows], right[rows]), s
    for s, length in ((0, 64 * which["width"] + 1), (1, -1), (1, -2 ** 31), (0, 2 ** 31 - 1)):
        lengths = b.lengths.copy()
        lengths[s] = length
        be.write(b.seqs.lengths, lengths)
        others([s])
    be.write(b.seqs.lengths, b.lengths)
    starts = b.starts.copy()
    starts[1] = b.rows + 3  # the first leaves the rows, the second ends before it begins
    be.write(b.seqs.starts, starts)
    others([0, 1])
    starts[:2] = -1, b.starts[1]  # the first begins before the rows
    be.write(b.seqs.starts, starts)
    others([0])
    b.free()
