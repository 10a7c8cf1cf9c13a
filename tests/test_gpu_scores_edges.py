"""Logits rows at the edges of what the scores and losses take: against 64 bits, tolerances as in
tests/scores_reference.py where no other bound is worked out beside the test."""
import math

import numpy as np
import pytest
import torch

from promptboot_amd import sampler as s
from promptboot_amd.scores import RowScorer
from tests import scores_reference as ref
from tests.test_gpu_scores import DEV, TYPES, make_logits, near, out, read_errors, records

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def scorer():
    sc = RowScorer(0)
    yield sc
    sc.close()


def distill_rest(x, ids, logit, T, lse, w):
    """The distillation with a rest bucket by logarithms of the masses: (loss, gradient, bound of the gradient before
    its rounding).

    The bound: with tol the error of a log-sum (of the row, or of what is off the list), a listed element's q and
    an off-list element's share of the rest are within 2 tol of themselves, relatively, and so is the student's mass
    off the list."""
    y = x.double() / T
    rows = torch.arange(x.shape[0], device=x.device)[:, None]
    listed = torch.zeros(y.shape, dtype=torch.bool, device=x.device)
    listed[rows, ids] = True
    own = torch.logsumexp(y, 1)
    rest = torch.logsumexp(y.masked_fill(listed, -math.inf), 1)
    log_qr = rest - own
    p = torch.exp(logit.double() / T - lse.double()[:, None])
    left = (1.0 - p.sum(1)).clamp(min=0.0)
    mass = p.sum(1) + left
    loss = (p * (torch.log(p) - (y - own[:, None]).gather(1, ids))).sum(1)
    loss = loss + torch.where(left > 0.0, left * (torch.log(left) - log_qr), 0.0)
    dense = torch.zeros_like(y).scatter_(1, ids, p)
    q, share = torch.exp(y - own[:, None]), torch.exp(y - rest[:, None])
    qr = torch.exp(log_qr)
    grad = torch.where(listed, mass[:, None] * q - dense, share * (mass * qr - left)[:, None])
    big = torch.where(torch.isfinite(y), y.abs(), 0.0).amax(1)
    tol = 2.0 * ref.EPS32 * (3.0 * big + 104.0)
    bound = torch.where(listed, mass[:, None] * q, share * (2.0 * mass * qr + left)[:, None]) * 2.0 * tol[:, None]
    scale = (w.double() / T)[:, None]
    return loss, grad * scale, bound * scale.abs(), tol


def listed_in(ids, n):
    """Which of the first n ids are in `ids`."""
    return (ids[:, None] == torch.arange(n, device=ids.device)).any(0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(70, 1_000), (1_100, 300), (2, 100_003), (64, 20_011)])
@pytest.mark.parametrize("T,gap", [(1.0, 80.0), (1.0, 88.0), (1.0, 110.0), (1.0, 400.0), (1.0, 740.0), (1.0, 1_000.0),
                                   (2.0, 20_000.0), (0.01, 1.5), (0.05, 7.0), (0.3, 30.0)])
def test_a_rest_of_little_mass_keeps_its_gradient(scorer, rows, vocab, dtype, T, gap):
    """Off-list logits `gap` below the listed ones: the teacher's remaining mass still pulls them up."""
    k = 10
    x, g = make_logits(rows, vocab, dtype, seed=vocab + int(gap), spread=0.5)
    x.clamp_(max=1.0).sub_(gap)
    ids = torch.topk(torch.rand((rows, vocab), generator=g, device=DEV), k, dim=1).indices
    x.scatter_(1, ids, (10.0 + torch.randn((rows, k), generator=g, device=DEV) * T).to(x.dtype))
    x[0, :3] = torch.where(listed_in(ids[0], 3), x[0, :3], -math.inf)  # some ids are excluded altogether
    logit = torch.randn((rows, k), generator=g, device=DEV) * T
    left = torch.rand(rows, generator=g, device=DEV) * 0.3
    left[rows // 2:] *= 1e-4
    lse = (torch.logsumexp(logit.double() / T, 1) - torch.log1p(-left.double())).float()
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    loss, grad, err = out(rows), torch.full_like(x, 5.0), records(rows)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse, weight=w, loss=loss, grad=grad, err=err, temperature=T)
    assert not read_errors(err).view(np.uint8).any()
    want, want_grad, bound, tol = distill_rest(x, ids, logit, T, lse, w)
    near(loss, want, ref.scalar_tolerance(want, 2 * tol), "loss")
    info = torch.finfo(x.dtype)
    half = info.eps / 2
    # an exponential below 2^-126 (1.2e-38) counts 0, times a factor of at most 1.3 w / T
    lost = 2e-38 * (1.0 + w.double() / T)[:, None]
    near(grad, want_grad, half * want_grad.abs() + bound * (1 + half) + float(info.tiny) * info.eps + lost, "grad")


@pytest.mark.parametrize("smooth", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("masked", ["chosen", "rejected"])
def test_a_token_without_weight_in_a_pair(scorer, masked, smooth):
    """A -inf logit at a token makes the margin infinite: sigma of it is 1 or 0, and a term of factor 0 counts 0."""
    vocab, beta, T = 300, 0.2, 0.7
    x, g = make_logits(8, vocab, "f32", seed=5)
    token = torch.randint(0, vocab, (8,), generator=g, device=DEV)
    row = 1 if masked == "chosen" else 3
    x[row, token[row]] = -math.inf
    start = torch.tensor([0, 2, 4, 6, 8], dtype=torch.int32, device=DEV)
    loss, logprob, grad, err = out(2), out(4), out(8, vocab), records(2)
    scorer.preference_loss(x, token.int(), start, beta=beta, label_smoothing=smooth, loss=loss, logprob=logprob,
                           grad=grad, err=err, temperature=T)
    assert not read_errors(err).view(np.uint8).any()
    factor = 1.0 - smooth if masked == "chosen" else smooth  # of the term that is infinite
    assert loss[0] == (math.inf if factor > 0.0 else 0.0) and torch.isfinite(loss[1])
    assert logprob[row // 2] == -math.inf and torch.isfinite(logprob[[1 - row // 2, 2, 3]]).all()
    slope = (smooth if masked == "rejected" else smooth - 1.0) * beta / T
    q = torch.softmax(x[:4].double() / T, 1)
    one = torch.zeros_like(q).scatter_(1, token[:4, None], 1.0)
    side = torch.tensor([1.0, 1.0, -1.0, -1.0], dtype=torch.float64, device=DEV)[:, None]
    want = slope * side * (one - q)
    tol = 2.0 * ref.lse_tolerance(x[:4], T)[:, None]
    near(grad[:4], want, ref.grad_tolerance(want, abs(slope), q, tol, x.dtype) + abs(slope) * one * q * tol, "grad")
    assert torch.isfinite(grad[4:]).all() and (grad[4:] != 0).any()


def long_tolerance(y, per):
    """ref.lse_tolerance for a thread's 768 terms, the most that are added in 32 bits: 768 / `per` sums of a chunk."""
    return ref.EPS32 * (3.0 * y + 8.0 + 768 / per)


def test_long_rows_are_not_summed_in_32_bits(scorer):
    """The longest rows: every thread rounds the same way where all of its terms are alike."""
    rows, vocab, low = 64, 4_194_304, 0.6785145998001099
    x = torch.full((rows, vocab), -low, device=DEV)
    x[:, :4096] = 0.0
    token = torch.arange(rows, dtype=torch.int32, device=DEV) * 60_000
    weigh = 4096.0 + (vocab - 4096) * math.exp(-low)
    lse = math.log(weigh)
    lp, loss, kl = out(rows), out(rows), out(rows)
    grad = torch.full_like(x, 5.0)
    own = x.gather(1, token.long()[:, None])[:, 0].double() - lse
    scorer.policy_loss(x, token, own.float(), torch.ones(rows, device=DEV), loss=loss, logprob=lp, kl=kl, grad=grad)
    tol = long_tolerance(low, 4)
    near(lp, own, ref.scalar_tolerance(own, torch.full((rows,), 2 * tol, device=DEV)), "logprob")
    # 1 / T times the ratio, which is 1 up to the rounding of the old log-probability and the error of the new
    ratio = torch.exp(own - own.float().double())
    want = (ratio / weigh * math.exp(-low))[:, None]
    grad.scatter_(1, token.long()[:, None], want.float())
    near(grad[:, 4096:].amin(1, keepdim=True), want, want * (4 * tol + 8 * ref.EPS32), "least gradient")
    near(grad[:, 4096:].amax(1, keepdim=True), want, want * (4 * tol + 8 * ref.EPS32), "largest gradient")
    few = torch.full((rows, 1), 7.0, device=DEV)
    scorer.distill_loss(x, token[:, None], few, loss=loss, lse=lp, grad=grad)
    want_lse = torch.full((rows,), lse, dtype=torch.float64, device=DEV)
    near(lp, want_lse, ref.scalar_tolerance(want_lse, torch.full((rows,), tol, device=DEV)), "lse")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(66, 393_216), (66, 393_219), (300, 393_217), (64, 786_433), (3, 1_048_579)])
def test_rows_around_the_longest_of_one_workgroup(scorer, rows, vocab, dtype):
    k, T, per = 40, 0.7, 4 if dtype == "f32" else 8
    x, g = make_logits(rows, vocab, dtype, seed=vocab, pad=1)
    ids = torch.linspace(0, vocab - 1, k, device=DEV).long().repeat(rows, 1)
    logit = torch.randn((rows, k), generator=g, device=DEV)
    lse = (torch.logsumexp(logit.double() / T, 1) + 0.2).float()
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    loss, grad = out(rows), torch.full_like(x, 5.0)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse, weight=w, loss=loss, grad=grad, temperature=T)
    half = torch.finfo(x.dtype).eps / 2
    for lo in range(0, rows, 32):
        r = slice(lo, lo + 32)
        want, want_grad, bound, _ = distill_rest(x[r], ids[r], logit[r], T, lse[r], w[r])
        tol = long_tolerance(x[r].double().abs().amax(1) / T, per)
        near(loss[r], want, ref.scalar_tolerance(want, 2 * tol), "loss")
        bound = bound / (2.0 * ref.EPS32 * (3.0 * x[r].double().abs().amax(1) / T + 104.0))[:, None] * 2.0 * tol[:, None]
        near(grad[r], want_grad, half * want_grad.abs() + bound * (1 + half) + 1e-36, "grad")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(2, 100_003), (40, 20_011), (1_100, 9_001)])
@pytest.mark.parametrize("gap", [15.0, 24.0, 45.0, 64.0])
def test_saturated_rows_have_no_probability_above_one(scorer, rows, vocab, dtype, gap):
    """One token holds all of a row's mass, `gap` above everything that its thread has met before it.

    Its exponent keeps the place of 16: it is off by 2^-21, 2^a by ln 2 times that and 3 roundings of its own, and
    nothing else is in the sum.  The moment's product e a has two roundings more, of at most 16.  (About a shift that
    stays 64 / T ln 2 = 132 below, a alone is off by 2^-17: 5e-6 in the log-probability, 8e-5 in the entropy.)"""
    T = 0.7
    x, g = make_logits(rows, vocab, dtype, seed=vocab, spread=0.5)
    x.clamp_(max=1.0)
    token = vocab - 1 - torch.randint(0, vocab // 5, (rows,), generator=g, device=DEV)
    top = gap + 2.0 + torch.rand((rows, 1), generator=g, device=DEV) * 3.0
    x.scatter_(1, token[:, None], top.to(x.dtype))
    want = ref.logprobs(x, token, T)
    tol = 2.0 ** -21 * math.log(2) + 3 * ref.EPS32
    tol_entropy = tol + math.log(2) * (2.0 ** -21 + 2 * 16 * ref.EPS32)
    lp, ent, lse, loss = out(rows), out(rows), out(rows), out(rows)
    value, ids = out(rows, 1), out(rows, 1, dtype=torch.int32, fill=0)

    def check(what):
        near(lp, want["logprob"], ref.scalar_tolerance(want["logprob"], torch.full_like(want["lse"], tol)), what)

    def check_lse(what):
        near(lse, want["lse"], ref.scalar_tolerance(want["lse"], torch.full_like(want["lse"], tol)), what)

    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, temperature=T)
    check("logprob"), check_lse("lse")
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, entropy=ent, temperature=T)
    check("logprob beside the entropy"), check_lse("lse beside the entropy")
    near(ent, want["entropy"], ref.scalar_tolerance(want["entropy"], torch.full_like(want["lse"], tol_entropy)), "entropy")
    scorer.top_logits(x, 1, token=ids, value=value, lse=lse, temperature=T)
    check_lse("lse of the top logits")
    zero, grad = torch.zeros(rows, device=DEV), torch.empty_like(x)
    scorer.policy_loss(x, token.int(), zero, zero, loss=loss, logprob=lp, temperature=T)
    check("policy")
    scorer.policy_loss(x, token.int(), zero, zero, loss=loss, logprob=lp, grad=grad, temperature=T)
    check("policy with its gradient")
    one = torch.zeros((rows, 1), device=DEV)
    for rest in (None, zero + 0.1):
        scorer.distill_loss(x, token.int()[:, None], one, teacher_lse=rest, loss=loss, lse=lse, grad=grad, temperature=T)
        check_lse("distillation")
    start = torch.arange(rows + 1, dtype=torch.int32, device=DEV)
    scorer.preference_loss(x, token.int(), start, beta=0.1, loss=loss, logprob=lp, temperature=T)
    check("preference")


@pytest.mark.parametrize("rows,vocab", [(4, 33), (1_100, 40), (3, 9_001)])
@pytest.mark.parametrize("offset", [0.0, 300.0, -2_000.0])
def test_a_log_sum_in_two_words_gives_exact_gradients(scorer, rows, vocab, offset):
    """q = 2^(x c - log-sum), T = 1: c is off by 1.3e-8 of itself, which leaves 1.3e-8 |ln q| (the log-sum is off with
    it); the exponent is a fused multiply-add, off by 2^-24 of itself; the sums of at most 9,001 / 256 / 4 + 1 chunks
    of four have 10 + 3 + 2 roundings; 2^a, alpha, beta, their sum and product 6.  Weights under 2^-24 of the row's
    largest count by their share alone.  lse alone is off by half a step of itself, 1.5e-5 at 300."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn((rows, vocab), generator=g, device=DEV) * 2.5 + offset
    token = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    gl, ge = torch.randn(rows, generator=g, device=DEV), torch.randn(rows, generator=g, device=DEV) * 0.1
    lp, lse, low, ent = out(rows), out(rows), out(rows), out(rows)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, lse_low=low, entropy=ent)
    want = ref.logprobs(x, token)
    tol = ref.EPS32 * (10 + 3 + 2 + 6 + 24) + 24 * 1.3e-8
    both = lse.double() + low.double()
    near(both, want["lse"], tol + 1.3e-8 * want["lse"].abs(), "the log-sum")
    assert (low.abs() <= 1.01 * ref.EPS32 * lse.abs() + 1e-12).all()
    q = torch.softmax(x.double(), 1)
    log_q = (x.double() - want["lse"][:, None])
    for a, b in ((gl, None), (gl, ge)):
        grad = out(rows, vocab)
        kw = {} if b is None else dict(grad_entropy=b, entropy=ent)
        scorer.token_logprobs_grad(x, token.int(), lse, lse_low=low, grad=grad, grad_logprob=a, **kw)
        zero = torch.zeros_like(a)
        want_grad = ref.logprobs_grad(x, token, a, zero if b is None else b)
        scale = a.double().abs()[:, None]
        if b is not None:  # ln q + H is off by its own roundings beside those of q
            scale = scale + b.double().abs()[:, None] * (log_q.abs() + want["entropy"][:, None].abs() + 3.0)
        near(grad, want_grad, ref.EPS32 * want_grad.abs() + scale * q * tol + 1e-37, "gradient")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [5, 1_100])
def test_gradients_of_very_large_logits(scorer, rows, dtype):
    """Three equal logits of 60,000 at T = 0.01: their log-sum's nearest binary32 is up to a half away, and each has a
    third of the mass all the same, up to a handful of roundings."""
    vocab, T = 700, 0.01
    x, g = make_logits(rows, vocab, dtype, seed=rows)
    where = torch.topk(torch.rand((rows, vocab), generator=g, device=DEV), 3, dim=1).indices
    level = 50_000.0 + torch.arange(rows, device=DEV) % 10 * 1_024.0
    x.scatter_(1, where, level[:, None].expand(-1, 3).to(x.dtype))
    token = where[:, 0]
    want = torch.zeros((rows, vocab), dtype=torch.float64, device=DEV)
    want.scatter_(1, where, torch.tensor([2.0, -1.0, -1.0], dtype=torch.float64, device=DEV).expand(rows, 3) / 3 / T)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 12 * ref.EPS32 * want.abs() + 1e-30
    lp, lse, low, one = out(rows), out(rows), out(rows), torch.ones(rows, device=DEV)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, lse_low=low, temperature=T)
    third = torch.full((rows,), -math.log(3.0), dtype=torch.float64, device=DEV)
    near(lp, third, ref.scalar_tolerance(third, torch.full((rows,), 6 * ref.EPS32, device=DEV)), "logprob")
    grad = torch.full_like(x, 5.0)
    scorer.token_logprobs_grad(x, token.int(), lse, lse_low=low, grad=grad, grad_logprob=one, temperature=T)
    near(grad, want, tol, "log-probability")
    scorer.policy_loss(x, token.int(), lp, one, loss=out(rows), grad=grad, temperature=T)
    near(grad, -want, tol, "policy")
    scorer.distill_loss(x, where.int()[:, :1].contiguous(), one[:, None], loss=out(rows), grad=grad, temperature=T)
    near(grad, -want, tol, "distillation")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(3, 60_001), (70, 1_003), (1_100, 301)])
def test_gradients_between_the_rows_of_the_logits(scorer, rows, vocab, dtype):
    """Logits and gradient as columns of one buffer, and as its even and odd rows."""
    x, g = make_logits(rows, vocab, dtype, seed=vocab)
    token = torch.randint(0, vocab, (rows,), generator=g, device=DEV).int()
    one, lse = torch.ones(rows, device=DEV), out(rows)
    ids, logit = token[:, None].contiguous(), torch.zeros((rows, 1), device=DEV)
    start = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=DEV)
    scorer.token_logprobs(x, token, logprob=out(rows), lse=lse)

    def calls(y, grad):
        scorer.policy_loss(y, token, -one, one, loss=out(rows), grad=grad)
        yield
        scorer.distill_loss(y, ids, logit, loss=out(rows), grad=grad)
        yield
        scorer.preference_loss(y, token, start, beta=0.1, loss=out(1), grad=grad)
        yield
        scorer.token_logprobs_grad(y, token, lse, grad=grad, grad_logprob=one)
        yield

    beside = torch.full((rows, 2 * vocab + 3), 5.0, dtype=x.dtype, device=DEV)
    between = torch.full((2 * rows, vocab + 1), 5.0, dtype=x.dtype, device=DEV)
    apart = torch.empty_like(x)
    for y, grad, rest in ((beside[:, :vocab], beside[:, vocab + 1:2 * vocab + 1], beside),
                          (between[::2, :vocab], between[1::2, :vocab], between)):
        y.copy_(x)
        for _ in zip(calls(x, apart), calls(y, grad)):
            assert torch.equal(grad, apart) and torch.equal(y, x)
        grad.fill_(5.0), y.fill_(5.0)
        assert (rest == 5.0).all()


@pytest.mark.parametrize("rows,vocab", [(4, 500), (4, 151_936), (1_100, 300)])
def test_a_policy_token_without_weight(scorer, rows, vocab):
    """ln q = -inf: the ratio is 0, and exp(d) - d - 1 grows without bound with d."""
    x, g = make_logits(rows, vocab, "f32", seed=vocab)
    token = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    x.scatter_(1, token[:, None], -math.inf)
    adv = torch.where(torch.arange(rows, device=DEV) % 2 == 0, 2.0, -2.0)
    old, r = torch.full((rows,), -3.0, device=DEV), torch.full((rows,), -2.0, device=DEV)
    for coef in (0.0, 0.1):
        for grad in (None, torch.full_like(x, 5.0)):
            loss, lp, kl, err = out(rows), out(rows), out(rows), records(rows)
            scorer.policy_loss(x, token.int(), old, adv, ref_logprob=r, kl_coef=coef, loss=loss, logprob=lp, kl=kl,
                               grad=grad, err=err)
            assert not read_errors(err).view(np.uint8).any()
            assert (lp == -math.inf).all() and (kl == math.inf).all()
            if coef != 0.0:
                assert (loss == math.inf).all()
                continue
            want = torch.where(adv > 0, 0.0, 1.6)  # the surrogate alone
            near(loss, want, torch.full_like(want, 1e-6), "loss")
            if grad is not None:  # an open ratio of 0 has a slope of 0
                assert (grad == 0).all()


def test_many_long_rows_behind_separate_reservations():
    sc = RowScorer(0)
    sc.reserve(2_000, 100)
    sc.reserve(2, 5_000)
    x, g = make_logits(2_000, 5_000, "bf16", seed=1)
    token = torch.randint(0, 5_000, (2_000,), generator=g, device=DEV)
    lp = out(2_000)
    sc.token_logprobs(x, token.int(), logprob=lp)
    want = ref.logprobs(x, token)["logprob"]
    near(lp, want, ref.scalar_tolerance(want, 2 * ref.lse_tolerance(x, 1.0)), "logprob")
    sc.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(2, 100_003), (40, 20_011), (1_100, 9_001)])
@pytest.mark.parametrize("level", [-8.0, -15.0, -25.0, -40.0])
def test_masked_first_chunks_cost_no_precision(scorer, rows, vocab, dtype, level):
    """All of a row is masked but one token below 0: its thread has met nothing to take a shift from.

    A sum of at least 2^-16 is kept about 0: the exponent has the place of 16 and is off by 2^-21, as in the test of
    saturated rows.  (Kept down to 2^-60 it was off by 2^-19: 1.3e-6 in the log-probability.)"""
    T = 0.7
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.full((rows, vocab), -math.inf, device=DEV).to(torch.float32)
    token = vocab - 1 - torch.randint(0, vocab // 5, (rows,), generator=g, device=DEV)
    x.scatter_(1, token[:, None], level - torch.rand((rows, 1), generator=g, device=DEV) * 4.0)
    x = x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    want_lse = x.gather(1, token[:, None])[:, 0].double() / T
    tol = 2.0 ** -21 * math.log(2) + 3 * ref.EPS32
    tol_lse = torch.full_like(want_lse, tol) + 2 * ref.EPS32 * want_lse.abs()  # c is rounded
    zero = torch.zeros(rows, device=DEV)
    lp, ent, lse, loss, grad = out(rows), out(rows), out(rows), out(rows), torch.empty_like(x)

    def check(what):
        near(lp, zero, torch.full_like(want_lse, tol), what)

    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, entropy=ent, temperature=T)
    check("logprob")
    near(lse, want_lse, ref.scalar_tolerance(want_lse, tol_lse), "lse")
    near(ent, zero, torch.full_like(want_lse, tol + math.log(2) * (2.0 ** -21 + 2 * 16 * ref.EPS32)), "entropy")
    scorer.top_logits(x, 1, token=out(rows, 1, dtype=torch.int32, fill=0), value=out(rows, 1), lse=lse, temperature=T)
    near(lse, want_lse, ref.scalar_tolerance(want_lse, tol_lse), "lse of the top logits")
    for kw in ({}, dict(grad=grad)):
        scorer.policy_loss(x, token.int(), zero, zero, loss=loss, logprob=lp, temperature=T, **kw)
        check("policy")
    start = torch.arange(rows + 1, dtype=torch.int32, device=DEV)
    scorer.preference_loss(x, token.int(), start, beta=0.1, loss=loss, logprob=lp, temperature=T)
    check("preference")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(2, 473), (3, 100_003), (70, 9_001), (1_100, 300)])
@pytest.mark.parametrize("T", [0.5, 1.0, 1.5, 2.0, 10.0, 100.0])
def test_finite_masks_weigh_nothing(scorer, rows, vocab, T, dtype):
    """-1e9 and less down to the type's lowest value, over whole chunks, threads and parts, at temperatures that keep
    them in binary32's range."""
    lowest = torch.finfo(TYPES[dtype]).min
    levels = torch.tensor([-1e9, -1e10, -3e15, -1e30, lowest], device=DEV)
    x, g = make_logits(rows, vocab, dtype, seed=vocab)
    r = torch.arange(rows, device=DEV)
    col = torch.arange(vocab, device=DEV)[None, :]
    keep = torch.randint(0, vocab, (rows, 1), generator=g, device=DEV)
    scattered = torch.rand((rows, vocab), generator=g, device=DEV) < 0.7
    masked = torch.where((r % 3 == 0)[:, None], col < vocab // 2, torch.where((r % 3 == 1)[:, None], scattered, col != keep))
    masked &= col != keep
    x.copy_(torch.where(masked, levels[r % 5][:, None], x.float()))
    clean = torch.where(masked, -math.inf, x.double())  # what a mask of -inf would leave
    token = keep[:, 0]
    want = ref.logprobs(clean, token, T)
    y = clean / T
    tol = ref.EPS32 * (3 * torch.where(torch.isfinite(y), y.abs(), 0.0).amax(1) + 8 + 192)
    lp, lse, low, ent, loss, err = out(rows), out(rows), out(rows), out(rows), out(rows), records(rows)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, lse_low=low, entropy=ent, err=err, temperature=T)
    assert not read_errors(err).view(np.uint8).any()
    near(lp, want["logprob"], ref.scalar_tolerance(want["logprob"], 2 * tol), "logprob")
    near(lse, want["lse"], ref.scalar_tolerance(want["lse"], tol), "lse")
    near(ent, want["entropy"], ref.scalar_tolerance(want["entropy"], 4 * tol), "entropy")
    one, grad = torch.ones(rows, device=DEV), torch.full_like(x, 5.0)
    q = torch.softmax(y, 1)
    delta = torch.zeros_like(q).scatter_(1, token[:, None], 1.0)
    half = torch.finfo(x.dtype).eps / 2

    def check(sign, what):
        bound = (half * (delta - q).abs() + 4 * tol[:, None] * (q + (delta - q).abs())) / T + 1e-36
        near(grad, sign * (delta - q) / T, bound, what)
        assert (grad[masked] == 0).all(), what

    scorer.token_logprobs_grad(x, token.int(), lse, lse_low=low, grad=grad, grad_logprob=one, temperature=T)
    check(1.0, "log-probability")
    scorer.policy_loss(x, token.int(), lp, one, loss=loss, grad=grad, err=err, temperature=T)
    assert not read_errors(err).view(np.uint8).any()
    check(-1.0, "policy")
    zero = torch.zeros((rows, 1), device=DEV)
    scorer.distill_loss(x, token.int()[:, None], zero, loss=loss, lse=lse, grad=grad, err=err, temperature=T)
    assert not read_errors(err).view(np.uint8).any()
    check(-1.0, "distillation")
    near(loss, -want["logprob"], ref.scalar_tolerance(want["logprob"], 2 * tol), "distillation")
    scorer.top_logits(x, 1, token=out(rows, 1, dtype=torch.int32, fill=0), value=out(rows, 1), lse=lse, err=err,
                      temperature=T)
    assert not read_errors(err).view(np.uint8).any()
    near(lse, want["lse"], ref.scalar_tolerance(want["lse"], tol), "lse of the top logits")


def test_rows_of_one_finite_mask(scorer):
    """Up to 2^31 in y / ln 2 a row of equal logits is the uniform distribution; past it nothing weighs, or the row
    fails at its first such logit."""
    vocab = 3_001
    for level, ok in [(-1e9, True), (-1.4e9, True), (1.4e9, True), (-1.6e9, False), (1.6e9, False), (-1e12, False),
                      (1e12, False), (3e15, False), (-1e30, False), (1e30, False)]:
        for rows in (2, 70):
            x = torch.full((rows, vocab), level, device=DEV)
            token = torch.arange(rows, dtype=torch.int32, device=DEV) * 7
            lp, ent, loss, err = out(rows), out(rows), out(rows), records(rows)
            grad = torch.full_like(x, 5.0)
            scorer.token_logprobs(x, token, logprob=lp, entropy=ent, err=err)
            e = read_errors(err)
            scorer.policy_loss(x, token, torch.full_like(lp, -math.log(vocab)), torch.ones_like(lp), loss=loss, grad=grad)
            if ok:
                assert not e.view(np.uint8).any(), level
                want = torch.full((rows,), -math.log(vocab), dtype=torch.float64, device=DEV)
                near(lp, want, torch.full_like(want, 4e-6), "logprob")  # 12 sums of a chunk and 3 roundings: 2e-6
                near(ent, -want, torch.full_like(want, 1.2e-5), "entropy")  # and a moment about up to 2^6
                other = grad[:, -1].double() * vocab
                near(other, torch.ones_like(want), torch.full_like(want, 2e-5), "gradient")
            else:
                assert (e["status"] == s.NONFINITE_OUTPUT).all() and not e["detail"].astype(np.uint32).any(), level
                assert lp.isnan().all() and loss.isnan().all() and grad.isnan().all()
