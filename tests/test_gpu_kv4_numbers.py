"""The attention and norm tests of a 4-bit cache once more, where a result that
is no number fails: their own comparison asks whether an error is above its
bound, which NaN is not. No counterpart in the reference."""
import itertools

import numpy as np
import pytest

import kv4_plain as plain
import test_gpu_kv4 as tokens
import test_gpu_kv4_prompts as prompts
from kv4_compare import expect

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be(backend):
    yield backend


def cases(test):
    """The arguments that a test is called with, by its parametrize marks."""
    axes = []
    for mark in getattr(test, "pytestmark", []):
        names = [n.strip() for n in mark.args[0].split(",")]
        axes.append([dict(zip(names, v if len(names) > 1 else (v,))) for v in mark.args[1]])
    for some in itertools.product(*axes):
        kw = {k: v for part in some for k, v in part.items()}
        yield pytest.param(test, kw, id="%s-%s" % (test.__name__[5:], "-".join(str(v) for v in kw.values())))


COMPARED = [tokens.test_attention, tokens.test_window, tokens.test_views_and_gate, tokens.test_captured_and_replayed,
            tokens.test_more_sequences_than_a_wave, prompts.test_attention, prompts.test_window, prompts.test_views_and_gate,
            prompts.test_few_rows_in_pieces, prompts.test_a_prompt_among_single_tokens]


@pytest.mark.parametrize("test,kw", [c for t in COMPARED for c in cases(t)])
def test_attention_gives_numbers(be, monkeypatch, test, kw):
    monkeypatch.setattr(tokens, "check", expect)
    monkeypatch.setattr(prompts, "check", expect)
    test(be, **kw)


@pytest.mark.parametrize("test,kw", list(cases(tokens.test_norm_rope)))
def test_norms_are_numbers(be, monkeypatch, test, kw):
    taken = plain.from_bits

    def from_bits(raw, type):
        x = taken(raw, type)
        assert np.isfinite(x).all()
        return x
    monkeypatch.setattr(plain, "from_bits", from_bits)
    test(be, **kw)
