"""Refusals of the two-word log-sum (no GPU): every one comes before it."""
import ctypes

import pytest

from promptboot_amd import sampler as s
from promptboot_amd import scores

A = 1 << 20  # an address nobody reads


def forward(**kw):
    v = dict(logits=A, dtype=scores.F32, vocab=100, ld=128, rows=4, T=1.0, token=A, out=A, lse=A, low=A, ent=A, err=A)
    v.update(kw)
    e = s._Error()
    st = s.lib().pb_token_logprobs_wide(None, v["logits"], v["dtype"], v["vocab"], v["ld"], v["rows"], v["T"],
                                        v["token"], v["out"], v["lse"], v["low"], v["ent"], v["err"], None,
                                        ctypes.byref(e))
    return st, e


def backward(**kw):
    v = dict(logits=A, dtype=scores.F32, vocab=100, ld=128, rows=4, T=1.0, token=A, lse=A, low=A, ent=A, g=A, ge=A,
             grad=A + (1 << 16), grad_ld=128)
    v.update(kw)
    e = s._Error()
    st = s.lib().pb_token_logprobs_wide_grad(None, v["logits"], v["dtype"], v["vocab"], v["ld"], v["rows"], v["T"],
                                             v["token"], v["lse"], v["low"], v["ent"], v["g"], v["ge"], v["grad"],
                                             v["grad_ld"], None, ctypes.byref(e))
    return st, e


@pytest.mark.parametrize("call", [forward, backward])
def test_two_words_are_checked(call):
    for kw, status in [(dict(vocab=0), s.CAPACITY), (dict(ld=99), s.CAPACITY), (dict(T=0.0), s.ARITHMETIC),
                       (dict(low=A + 2), s.ALIGNMENT), (dict(lse=None), s.CAPACITY), (dict(logits=A + 2), s.ALIGNMENT),
                       (dict(token=None), s.CAPACITY)]:
        st, e = call(**kw)
        assert st == status and e.status == status, kw
    for kw in ({}, dict(low=None)):  # nothing is wrong but the missing context
        st, e = call(**kw)
        assert st == s.STATE and e.needed == 1
    assert call(rows=0)[0] == s.OK
    assert backward(grad=A)[0] == s.STATE and backward(grad=A + 4)[0] == s.STATE
