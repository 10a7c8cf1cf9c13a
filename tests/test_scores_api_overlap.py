"""Gradients that lie between the rows of their logits (no GPU)."""
import itertools

import pytest

from promptboot_amd import sampler as s
from promptboot_amd import scores
from tests.test_scores_api import A, WITH_GRAD, call


@pytest.mark.parametrize("name", WITH_GRAD)
def test_rows_between_each_other_are_no_overlap(name):
    for grad, ld, status in [
            (A + 100 * 4, 256, s.STATE), (A + 128 * 4, 256, s.STATE), (A + 156 * 4, 256, s.STATE),  # columns of one buffer
            (A - 128 * 4, 256, s.STATE), (A + (256 + 100) * 4, 256, s.STATE),
            (A + 99 * 4, 256, s.STATE), (A + 157 * 4, 256, s.STATE)]:
        st, e = call(name, ld=256, grad=grad, grad_ld=ld)
        off = (grad - A) // 4 % 256
        shared = off < 100 or off > 256 - 100
        assert st == status and (e.detail & 0xFFFFFFFF == 9) == shared, off
        assert (st == s.STATE and e.needed == 1) != shared  # the context is all that is missing


def test_every_small_layout_against_the_elements():
    """All offsets and strides of a few rows, element by element; two strides count by the ranges they span."""
    vocab = 3
    for rows, ld, gld, off in itertools.product((1, 2, 3), (3, 5, 7), (3, 5, 7), range(-24, 25)):
        a = {r * ld + j for r in range(rows) for j in range(vocab)}
        b = {off + r * gld + j for r in range(rows) for j in range(vocab)}
        want = bool(a & b) if ld == gld else not (max(a) < min(b) or max(b) < min(a))
        if off == 0 and ld == gld:
            want = False  # in place
        st, e = call("policy", dtype=scores.F32, vocab=vocab, ld=ld, rows=rows, grad=A + 4 * off, grad_ld=gld)
        assert st == s.STATE and (e.detail & 0xFFFFFFFF == 9) == want, (rows, ld, gld, off)
