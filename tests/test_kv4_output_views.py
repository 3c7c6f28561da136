"""The views that sm_kv4_read takes for its outputs, without a GPU: those
whose rows and heads do not overlap, rows first or heads first."""
import itertools

import pytest

import test_kv4_refusals as entries
from test_kv4_refusals import lib, view  # noqa: F401

BIG = {n: 1 << 50 for n in entries.READ.need}


def run(lib, stride, head, tokens, kv_heads):
    change = {"kv": view(stride, head, 3), "vv": None, "tokens": tokens, "longest": min(tokens, 4), "kv_heads": kv_heads}
    return entries.READ.run(lib, change=change, sizes=BIG)


def overlap(stride, head, tokens, heads, dim):
    first = sorted(t * stride + h * head for t, h in itertools.product(range(tokens), range(heads)))
    return any(b - a < dim for a, b in zip(first, first[1:]))


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 3), (5, 1), (5, 2), (3, 4)])
def test_rows_first_and_heads_first(lib, tokens, heads):  # noqa: F811
    dim = 72
    assert run(lib, heads * dim, dim, tokens, heads) == 0
    assert run(lib, dim, tokens * dim, tokens, heads) == 0  # as a cache of whole heads has them
    assert run(lib, dim + 5, (tokens - 1) * (dim + 5) + dim, tokens, heads) == 0
    if tokens > 1 and heads > 1:
        assert run(lib, dim + 5, (tokens - 1) * (dim + 5) + dim - 1, tokens, heads) == entries.ARG
        assert run(lib, dim - 1, 1000 * dim, tokens, heads) == entries.ARG
        assert run(lib, 1000 * dim, dim - 1, tokens, heads) == entries.ARG


def test_no_view_that_overlaps_is_taken(lib):  # noqa: F811
    dim = 72
    for tokens, heads in ((1, 1), (1, 2), (2, 1), (2, 2), (3, 4), (5, 3)):
        for stride, head in itertools.product(range(0, 6 * dim, 24), repeat=2):
            rc = run(lib, stride, head, tokens, heads)
            if overlap(stride, head, tokens, heads, dim):
                assert rc == entries.ARG, (stride, head, tokens, heads)
