"""Logits rows at the edges of what the scores and losses take: against 64 bits, tolerances as in
tests/scores_reference.py where no other bound is worked out beside the test."""
import math

import numpy as np
import pytest
import torch

from promptboot_amd.scores import RowScorer
from tests import scores_reference as ref
from tests.test_gpu_scores import DEV, make_logits, near, out, read_errors, records

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
