"""Refusals of the logits-row scores and losses, and their formulas' gradients against differences (no GPU)."""
import ctypes
import math

import pytest
import torch

from promptboot_amd import sampler as s
from promptboot_amd import scores
from tests import scores_reference as ref

A = 1 << 20  # an address nobody reads: every refusal comes before the GPU
ROWS = dict(logits=A, dtype=scores.F32, vocab=100, ld=128, rows=4, T=1.0)


def call(name, **kw):
    """A call without a context: (status, error record)."""
    v = dict(ROWS, k=5, token=A, out=A, lse=A, entropy=A, g=A, ge=A, grad=A + (1 << 16), grad_ld=128, tid=A, tlogit=A,
             tlse=A, w=A, old=A, adv=A, ref=A, low=0.2, high=0.2, kl=0.1, start=A, pairs=1, beta=0.1, smooth=0.0, err=A)
    v.update(kw)
    head = [None, v["logits"], v["dtype"], v["vocab"], v["ld"], v["rows"]]
    e = s._Error()
    tail = [None, ctypes.byref(e)]
    if name == "logprobs":
        args = [*head, v["T"], v["token"], v["out"], v["lse"], v["entropy"], v["err"], *tail]
    elif name == "logprobs_grad":
        args = [*head, v["T"], v["token"], v["lse"], v["entropy"], v["g"], v["ge"], v["grad"], v["grad_ld"], *tail]
    elif name == "top":
        args = [*head, v["k"], v["T"], v["token"], v["out"], v["lse"], v["err"], *tail]
    elif name == "distill":
        args = [*head, v["T"], v["k"], v["tid"], v["tlogit"], v["tlse"], v["w"], v["out"], v["lse"], v["grad"],
                v["grad_ld"], v["err"], *tail]
    elif name == "policy":
        args = [*head, v["T"], v["token"], v["old"], v["adv"], v["ref"], v["w"], v["low"], v["high"], v["kl"],
                v["out"], v["lse"], v["entropy"], v["grad"], v["grad_ld"], v["err"], *tail]
    else:
        args = [*head, v["T"], v["token"], v["start"], v["pairs"], v["ref"], v["w"], v["beta"], v["smooth"],
                v["out"], v["lse"], v["grad"], v["grad_ld"], v["err"], *tail]
    fn = dict(logprobs="pb_token_logprobs", logprobs_grad="pb_token_logprobs_grad", top="pb_top_logits",
              distill="pb_distill_loss", policy="pb_policy_loss", preference="pb_preference_loss")[name]
    return getattr(s.lib(), fn)(*args), e


NAMES = ["logprobs", "logprobs_grad", "top", "distill", "policy", "preference"]
WITH_GRAD = ["logprobs_grad", "distill", "policy", "preference"]


@pytest.mark.parametrize("name", NAMES)
def test_rows_are_checked(name):
    for kw, status in [
            (dict(vocab=0), s.CAPACITY), (dict(vocab=scores.SCORE_MAX_VOCAB + 1, ld=1 << 30), s.CAPACITY),
            (dict(rows=scores.SCORE_MAX_ROWS + 1), s.CAPACITY), (dict(ld=99), s.CAPACITY), (dict(ld=1 << 41), s.CAPACITY),
            (dict(dtype=3), s.STATE), (dict(T=0.0), s.ARITHMETIC), (dict(T=-1.0), s.ARITHMETIC),
            (dict(T=math.nan), s.ARITHMETIC), (dict(T=math.inf), s.ARITHMETIC), (dict(T=0.009), s.ARITHMETIC),
            (dict(logits=A + 2), s.ALIGNMENT), (dict(logits=A + 1, dtype=scores.BF16), s.ALIGNMENT),
            (dict(logits=None), s.CAPACITY)]:
        st, e = call(name, **kw)
        assert st == status and e.status == status, (kw, st)
    st, e = call(name)  # nothing else is wrong: the missing context is
    assert st == s.STATE and e.needed == 1
    assert call(name, rows=0, logits=None, token=None, out=None, grad=None, pairs=0)[0] == s.OK


@pytest.mark.parametrize("name", WITH_GRAD)
def test_gradients_are_checked(name):
    assert call(name, grad_ld=99)[0] == s.CAPACITY
    assert call(name, grad=A + (1 << 16) + 2)[0] == s.ALIGNMENT
    size = (3 * 128 + 100) * 4
    for grad, ld, status in [(A, 128, s.STATE), (A + 4, 128, s.STATE), (A + size - 4, 128, s.STATE),
                             (A, 129, s.STATE), (A + size, 128, s.STATE), (A - size + 4, 128, s.STATE)]:
        st, e = call(name, grad=grad, grad_ld=ld)
        overlap = e.detail & 0xFFFFFFFF == 9
        assert st == status and overlap == ((grad, ld) not in [(A, 128), (A + size, 128)]), (grad, ld)


@pytest.mark.parametrize("name,kw,status", [
    ("logprobs", dict(token=None), s.CAPACITY), ("logprobs", dict(out=None), s.CAPACITY),
    ("logprobs", dict(entropy=A + 2), s.ALIGNMENT), ("logprobs", dict(err=A + 4), s.ALIGNMENT),
    ("logprobs_grad", dict(lse=None), s.CAPACITY), ("logprobs_grad", dict(grad=None), s.CAPACITY),
    ("logprobs_grad", dict(entropy=None), s.CAPACITY),
    ("top", dict(k=0), s.CAPACITY), ("top", dict(k=101), s.CAPACITY), ("top", dict(k=129, vocab=128), s.CAPACITY),
    ("top", dict(token=None), s.CAPACITY),
    ("distill", dict(k=0), s.CAPACITY), ("distill", dict(k=129), s.CAPACITY), ("distill", dict(tid=None), s.CAPACITY),
    ("distill", dict(out=None), s.CAPACITY), ("distill", dict(tlogit=A + 1), s.ALIGNMENT),
    ("policy", dict(low=-0.1), s.ARITHMETIC), ("policy", dict(low=1.1), s.ARITHMETIC),
    ("policy", dict(high=-0.1), s.ARITHMETIC), ("policy", dict(high=math.nan), s.ARITHMETIC),
    ("policy", dict(kl=math.inf), s.ARITHMETIC), ("policy", dict(ref=None), s.CAPACITY),
    ("policy", dict(adv=None), s.CAPACITY), ("policy", dict(old=None), s.CAPACITY),
    ("preference", dict(beta=math.nan), s.ARITHMETIC), ("preference", dict(smooth=1.5), s.ARITHMETIC),
    ("preference", dict(start=None), s.CAPACITY), ("preference", dict(out=None), s.CAPACITY),
    ("preference", dict(pairs=scores.SCORE_MAX_ROWS + 1), s.CAPACITY)])
def test_arguments_are_checked(name, kw, status):
    st, e = call(name, **kw)
    assert st == status and e.status == status
    assert not (st == s.STATE and e.needed == 1)


def test_reservation_is_checked():
    fn = s.lib().pb_context_reserve_scores
    for rows, vocab, status in [(1, 0, s.CAPACITY), (1, scores.SCORE_MAX_VOCAB + 1, s.CAPACITY),
                                (scores.SCORE_MAX_ROWS + 1, 10, s.CAPACITY), (1, 10, s.STATE)]:
        e = s._Error()
        assert fn(None, rows, vocab, ctypes.byref(e)) == status and e.status == status


def test_header_constants():
    text = (s.LIB_PATH.parents[1] / "include" / "pbsample.h").read_text()
    for name in ("SCORE_MAX_ROWS", "SCORE_MAX_VOCAB", "TOP_LOGITS_MAX"):
        assert f"#define PB_{name} {getattr(scores, name)}u" in text


def test_buffers_on_the_host_are_refused():
    with pytest.raises(ValueError, match="lies on cpu"):
        scores._matrix(torch.zeros(2, 3), "logits", 0)
    x = torch.zeros(4, 6, device="meta")
    with pytest.raises(ValueError):
        scores._matrix(x.t(), "logits", 0)


class _Fake:
    """A buffer of another framework, on no device that it names."""

    def __init__(self, t):
        self.t, self.shape, self.dtype = t, t.shape, t.dtype

    def stride(self, i):
        return self.t.stride(i)

    def element_size(self):
        return self.t.element_size()

    def data_ptr(self):
        return self.t.data_ptr()


def test_rows_may_be_strided():
    t = torch.zeros(4, 10)
    assert scores._matrix(_Fake(t[:, :6]), "logits", 0)[1:] == (4, 6, 10)
    assert scores._matrix(_Fake(t[::2, 1:7]), "logits", 0)[1:] == (2, 6, 20)
    assert scores._matrix(_Fake(t[:1, :6]), "logits", 0)[1:] == (1, 6, 6)
    for bad in (t.t(), t[:, ::2], t[:1].expand(3, 10), t[0]):
        with pytest.raises(ValueError):
            scores._matrix(_Fake(bad), "logits", 0)
    for kind, code in ((torch.float32, scores.F32), (torch.bfloat16, scores.BF16), (torch.float16, scores.F16)):
        assert scores._dtype_of(_Fake(t.to(kind)), None) == code
    with pytest.raises(ValueError):
        scores._dtype_of(_Fake(t.double()), None)
    with pytest.raises(ValueError):
        scores._dtype_of(_Fake(t), "bf16")


# ---- the formulas ----

def differences(f, x, step=1e-6):
    """Central differences of a sum f by every element of x."""
    grad = torch.zeros_like(x)
    for i in range(x.shape[0]):
        for j in range(x.shape[1]):
            up, down = x.clone(), x.clone()
            up[i, j] += step
            down[i, j] -= step
            grad[i, j] = (f(up) - f(down)) / (2 * step)
    return grad


def test_gradients_against_differences():
    """The reference's gradients, which the kernels are held to, are those of the reference's losses."""
    g = torch.Generator().manual_seed(3)
    rows, vocab, k, T = 6, 9, 4, 1.7
    x = torch.randn((rows, vocab), generator=g, dtype=torch.float64) * 2
    token = torch.tensor([0, 8, 3, -1, 5, 2])
    a, b = (torch.randn(rows, generator=g, dtype=torch.float64) for _ in range(2))

    def near(got, want):
        assert (got - want).abs().max() < 1e-7

    def score(v):
        o = ref.logprobs(v, token, T)
        return (a * o["logprob"] + b * o["entropy"]).sum()

    near(ref.logprobs_grad(x, token, a, b, T), differences(score, x))
    ids = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    ids[1, 2] = ids[4, 0] = -1
    logit = torch.randn((rows, k), generator=g, dtype=torch.float64)
    w = torch.rand(rows, generator=g, dtype=torch.float64) + 0.5
    w[2] = 0.0
    lse = torch.logsumexp(torch.where(ids >= 0, logit / T, -math.inf), 1) + 0.3
    for tail in (None, lse):
        near(ref.distill(x, ids, logit, T, tail, w)["grad"],
             differences(lambda v: (w * ref.distill(v, ids, logit, T, tail, w)["loss"]).sum(), x))
    lp = ref.logprobs(x, token, T)["logprob"]
    old = lp - torch.log(torch.tensor([0.5, 1.5, 1.1, 1.0, 1.6, 0.7], dtype=torch.float64))
    r = lp + torch.randn(rows, generator=g, dtype=torch.float64) * 0.5
    args = (token, old, a, T, r, w, 0.2, 0.3, 0.4)
    near(ref.policy(x, *args)["grad"], differences(lambda v: (w * ref.policy(v, *args)["loss"]).sum(), x))
    start, pw = [0, 2, 3, 5, 6], torch.tensor([0.7, 1.3], dtype=torch.float64)
    r2 = torch.randn(4, generator=g, dtype=torch.float64)
    args = (token, start, 0.8, T, 0.1, r2, pw)
    near(ref.preference(x, *args)["grad"], differences(lambda v: (pw * ref.preference(v, *args)["loss"]).sum(), x))
