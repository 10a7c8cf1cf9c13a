"""Scores and losses of logits rows against the same in 64 bits, at the sizes, strides, types and masks where they
could go wrong.  Tolerances: tests/scores_reference.py."""
import math

import numpy as np
import pytest
import torch

from promptboot_amd import hip
from promptboot_amd import sampler as s
from promptboot_amd.scores import RowScorer
from tests import scores_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


@pytest.fixture(scope="module")
def scorer():
    sc = RowScorer(0)
    yield sc
    sc.close()


def make_logits(rows, vocab, dtype, seed=0, pad=0, shift=0, spread=2.5):
    """Rows of `vocab` + `pad` elements that start `shift` elements into their allocation; the rest is NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.full((rows * (vocab + pad) + shift + 8,), math.nan, dtype=TYPES[dtype], device=DEV)
    x = flat[shift:shift + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab]
    v = torch.randn((rows, vocab), generator=g, device=DEV) * spread
    if vocab > 8:
        v.scatter_add_(1, torch.randint(0, vocab, (rows, 3), generator=g, device=DEV),
                       torch.rand((rows, 3), generator=g, device=DEV) * 7 + 8)
    x.copy_(v)
    return x, g


def ids_of(x, g, masked=0.0):
    rows, vocab = x.shape
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    top = x.float().argmax(1)
    t = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.5, top, t)
    return torch.where(torch.rand(rows, generator=g, device=DEV) < masked, -1, t)


def out(*shape, dtype=torch.float32, fill=math.nan):
    return torch.full(shape, fill, dtype=dtype, device=DEV)


def records(rows):
    return torch.full((rows, 12), 77, dtype=torch.int32, device=DEV)


def read_errors(err):
    torch.cuda.synchronize()
    return err.cpu().numpy().view(s.ERROR_DTYPE).reshape(-1)


def near(got, want, tol, what):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan())
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][:3].tolist(),
                           want[bad][:3].tolist(), (tol.expand_as(got)[bad][:3]).tolist())


def near_grad(got, want, scale, x, T, tol, what="grad"):
    q = torch.softmax(x.double() / T, 1)
    near(got, want, ref.grad_tolerance(want, scale[:, None], q, tol[:, None], got.dtype), what)


# rows x vocab: single elements, a chunk's edges, many splits, one split, whole vocabularies
SHAPES = [(1, 1), (3, 2), (2, 7), (5, 8), (4, 9), (3, 63), (2, 64), (7, 65), (300, 33), (1, 1000), (40, 4099),
          (3, 32_768), (1100, 513), (2, 151_936), (9, 50_257)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_token_logprobs_and_gradient(scorer, rows, vocab, dtype):
    T = [1.0, 0.7, 2.0][(rows + vocab) % 3]
    x, g = make_logits(rows, vocab, dtype, seed=rows * vocab, pad=[0, 1, 5][rows % 3], shift=vocab % 5)
    token = ids_of(x, g, masked=0.2 if rows > 3 else 0.0)
    lp, lse, ent = out(rows), out(rows), out(rows)
    err = records(rows)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, entropy=ent, err=err, temperature=T)
    want = ref.logprobs(x, token, T)
    tol = ref.lse_tolerance(x, T)
    near(lse, want["lse"], ref.scalar_tolerance(want["lse"], tol), "lse")
    near(lp, want["logprob"], ref.scalar_tolerance(want["logprob"], 2 * tol), "logprob")
    # the moment has a further rounding per product and sum, of at most 100 per log2
    near(ent, want["entropy"], ref.scalar_tolerance(want["entropy"], 4 * tol), "entropy")
    assert not read_errors(err).view(np.uint8).any()
    gl = torch.randn(rows, generator=g, device=DEV)
    ge = torch.randn(rows, generator=g, device=DEV) * 0.1
    # lse and entropy come rounded: their half steps add to the weights' error
    tol = tol + ref.EPS32 * (want["lse"].abs() + want["entropy"].abs())
    q_range = 1.0 + (x.double() / T - want["lse"][:, None]).abs().amax(1) + want["entropy"]
    for gamma, eta in ((gl, ge), (gl, None), (None, ge)):
        full = torch.full((rows, vocab + 3), 5.0, dtype=x.dtype, device=DEV)
        grad = full[:, :vocab]
        scorer.token_logprobs_grad(x, token.int(), lse, grad=grad, grad_logprob=gamma, grad_entropy=eta,
                                   entropy=ent, temperature=T)
        zero = torch.zeros(rows, device=DEV)
        a, b = gl if gamma is not None else zero, ge if eta is not None else zero
        want_grad = ref.logprobs_grad(x, token, a, b, T)
        # the entropy's factor ln q + H multiplies the error, and has one of its own
        scale = (a.abs().double() + b.abs().double() * (q_range + 1.0)) / T
        near_grad(grad, want_grad, scale, x, T, tol)
        assert (full[:, vocab:] == 5.0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 7), (2, 64, 20), (4, 129, 128), (5, 1000, 1),
                                          (33, 4099, 64), (2, 151_936, 20), (300, 2000, 33), (1, 262_209, 128),
                                          (1030, 300, 128)])
def test_top_logits(scorer, rows, vocab, k, dtype):
    x, g = make_logits(rows, vocab, dtype, seed=vocab + k, pad=k % 3, shift=rows % 4)
    token, value, lse = out(rows, k, dtype=torch.int32, fill=9), out(rows, k), out(rows)
    scorer.top_logits(x, k, token=token, value=value, lse=lse, temperature=2.0)
    ids, values = ref.top(x, k)
    assert torch.equal(token.long(), ids)
    assert torch.equal(value.double(), values)
    want = torch.logsumexp(x.double() / 2.0, 1)
    near(lse, want, ref.scalar_tolerance(want, ref.lse_tolerance(x, 2.0)), "lse")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_top_logits_of_ties_and_masks(scorer, dtype):
    """Equal values everywhere, in a band, -0 beside 0, and rows masked but for fewer than k ids."""
    vocab, k = 5003, 50
    x, g = make_logits(6, vocab, dtype, seed=3)
    x[0] = 1.5
    x[1] = torch.round(x[1].float() / 4.0).to(x.dtype)
    x[2] = torch.where(torch.arange(vocab, device=DEV) % 3 == 0, -0.0, 0.0).to(x.dtype)
    x[3] = -math.inf
    x[3, 4000:4010] = 2.0
    x[4] = torch.finfo(x.dtype).min
    x[4, ::700] = -3.0
    x[5, 100:] = x[5, 99]
    token, value = out(6, k, dtype=torch.int32, fill=9), out(6, k)
    scorer.top_logits(x, k, token=token, value=value)
    ids, values = ref.top(x, k)
    assert torch.equal(token.long(), ids)
    assert torch.equal(value.double(), values)


def teacher(x, g, k, T, short=True):
    rows, vocab = x.shape
    ids = torch.topk(x.float() + torch.rand(x.shape, generator=g, device=DEV), k, dim=1).indices
    ids = ids[:, torch.randperm(k, generator=g, device=DEV)].contiguous()
    logit = x.gather(1, ids).float() + torch.randn((rows, k), generator=g, device=DEV)
    if short and k > 1:
        ids = torch.where(torch.rand((rows, k), generator=g, device=DEV) < 0.2, -1, ids)
        logit = torch.where(ids < 0, math.nan, logit)  # what stands beside padding is not looked at
    masked = torch.where(ids >= 0, logit.double(), -math.inf) / T
    lse = torch.logsumexp(masked, 1)
    left = torch.rand(rows, generator=g, device=DEV) * 0.3
    lse = torch.where(torch.isfinite(lse), lse, 0.0) - torch.log1p(-left.double())
    return ids, logit, lse.float()


def distill_scale(x, ids, logit, T, lse, w):
    """What multiplies an element's error of 2^a: the factors of q on and off the list."""
    y = x.double() / T
    q = torch.softmax(y, 1)
    valid = ids >= 0
    listed = torch.zeros_like(q).scatter_add_(1, ids.clamp(min=0), valid.double()) > 0
    rest = torch.where(listed, 0.0, q).sum(1)
    return (w.double().abs() / T) * (2.0 + torch.where(rest > 0, 1.0 / rest.clamp(min=1e-300), 0.0) * (lse is not None))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (2, 8, 5), (3, 65, 20), (70, 1000, 100), (5, 4099, 128),
                                          (2, 151_936, 20), (1100, 300, 7), (3, 262_209, 64)])
def test_distill_loss(scorer, rows, vocab, k, dtype, tail):
    T = [1.0, 2.0][k % 2]
    x, g = make_logits(rows, vocab, dtype, seed=vocab * k, pad=rows % 3, shift=k % 4)
    ids, logit, lse = teacher(x, g, k, T)
    if not tail:
        lse = None
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    w = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.2, 0.0, w)
    loss, own_lse, err = out(rows), out(rows), records(rows)
    full = torch.full((rows, vocab + 2), 5.0, dtype=x.dtype, device=DEV)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse, weight=w, loss=loss, lse=own_lse, grad=full[:, :vocab],
                        err=err, temperature=T)
    want = ref.distill(x, ids, logit, T, lse, w)
    tol = ref.lse_tolerance(x, T)
    assert not read_errors(err).view(np.uint8).any()
    near(own_lse, want["lse"], ref.scalar_tolerance(want["lse"], tol), "lse")
    near(loss, want["loss"], ref.scalar_tolerance(want["loss"], 2 * tol), "loss")
    near_grad(full[:, :vocab], want["grad"], distill_scale(x, ids, logit, T, lse, w), x, T, 2 * tol)
    assert (full[:, vocab:] == 5.0).all()
    # without a gradient the loss is the same up to the order of its sums: the same bound holds
    again = out(rows)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse, weight=w, loss=again, temperature=T)
    near(again, want["loss"], ref.scalar_tolerance(want["loss"], 2 * tol), "loss alone")


@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows_that_leave_nothing(scorer, tail):
    """Nothing listed, nothing listed that weighs, everything listed, the student masked off the list or on it."""
    vocab, k = 96, 96
    x, g = make_logits(5, vocab, "f32", seed=5)
    ids = torch.arange(vocab, device=DEV).repeat(5, 1)
    logit = torch.randn((5, k), generator=g, device=DEV)
    lse = torch.full((5,), 6.0, device=DEV)
    ids[0] = -1
    logit[1] = -math.inf
    lse[2] = torch.logsumexp(logit[2], 0)
    ids[3, 10:] = -1
    x[3, 10:] = -math.inf
    ids[4, 10:] = -1
    x[4, 3] = -math.inf  # a listed id of the teacher's that the student excludes
    loss, grad = out(5), out(5, vocab)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse if tail else None, loss=loss, grad=grad)
    want = ref.distill(x, ids, logit, 1.0, lse if tail else None)
    assert loss[0] == 0 and loss[1] == 0 and (grad[:2] == 0).all()
    assert loss[4] == math.inf and want["loss"][4] == math.inf
    tol = 2 * ref.lse_tolerance(x, 1.0)
    near(loss[:4], want["loss"][:4], ref.scalar_tolerance(want["loss"][:4], tol[:4]), "loss")
    scale = distill_scale(x, ids, logit, 1.0, lse if tail else None, torch.ones(5, device=DEV))
    near_grad(grad, want["grad"], scale, x, 1.0, tol)


@pytest.mark.parametrize("with_ref", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 9), (5, 64), (40, 1000), (2, 151_936), (1100, 257), (6, 50_257)])
def test_policy_loss(scorer, rows, vocab, dtype, with_ref):
    T = [1.0, 0.7][rows % 2]
    x, g = make_logits(rows, vocab, dtype, seed=rows + vocab, pad=rows % 4, shift=vocab % 3)
    token = ids_of(x, g, masked=0.2 if rows > 3 else 0.0)
    lp = ref.logprobs(x, token, T)["logprob"].float()
    # ratios from 0.6 to 1.6, none at a bound
    old = lp - torch.log(0.61 + torch.rand(rows, generator=g, device=DEV))
    adv = torch.randn(rows, generator=g, device=DEV)
    r = lp + torch.randn(rows, generator=g, device=DEV) * 0.3 if with_ref else None
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    w = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.1, 0.0, w)
    loss, logprob, kl, err = out(rows), out(rows), out(rows), records(rows)
    full = torch.full((rows, vocab + 1), 5.0, dtype=x.dtype, device=DEV)
    args = dict(ref_logprob=r, weight=w, clip_low=0.2, clip_high=0.28, kl_coef=0.1 if with_ref else 0.0, temperature=T)
    scorer.policy_loss(x, token.int(), old, adv, loss=loss, logprob=logprob, kl=kl, grad=full[:, :vocab], err=err,
                       **args)
    want = ref.policy(x, token, old, adv, T, r, w, 0.2, 0.28, 0.1 if with_ref else 0.0)
    assert not read_errors(err).view(np.uint8).any()
    tol = 2 * ref.lse_tolerance(x, T)
    near(logprob, want["logprob"], ref.scalar_tolerance(want["logprob"], tol), "logprob")
    gap = (r - lp).double().abs().exp() if with_ref else torch.zeros_like(tol)
    steep = 1.7 * adv.double().abs() + 0.1 * (gap + 1.0)
    near(kl, want["kl"], ref.scalar_tolerance(want["kl"], (gap + 1.0) * tol), "kl")
    near(loss, want["loss"], ref.scalar_tolerance(want["loss"], steep * tol), "loss")
    # (delta - q): the slope's own error goes with delta too
    live = (token >= 0) & (w != 0)
    q = torch.softmax(x.double() / T, 1)
    one = torch.zeros_like(q)
    one[live, token[live]] = 1.0
    bound = ref.grad_tolerance(want["grad"], (steep * w / T)[:, None], q, tol[:, None], x.dtype)
    bound = bound + (steep * w / T * tol)[:, None] * (one - q).abs() + want["slope"].abs()[:, None] * one * q * tol[:, None]
    near(full[:, :vocab], want["grad"], bound, "grad")
    assert (full[:, vocab:] == 5.0).all()


def test_policy_loss_branches(scorer):
    """Each side of each clip bound, with both signs of the advantage, and an advantage of 0."""
    vocab = 40
    x, g = make_logits(8, vocab, "f32", seed=11)
    token = ids_of(x, g)
    lp = ref.logprobs(x, token)["logprob"].float()
    ratio = torch.tensor([0.5, 0.5, 1.5, 1.5, 1.0, 1.0, 1.5, 1.1], device=DEV)
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0, 0.0, 2.0], device=DEV)
    loss, grad = out(8), out(8, vocab)
    scorer.policy_loss(x, token.int(), lp - torch.log(ratio), adv, loss=loss, grad=grad)
    torch.cuda.synchronize()
    moved = (grad != 0).any(1).tolist()
    assert moved == [True, False, False, True, True, True, False, True]
    want = torch.tensor([-0.5, 0.8, -1.2, 1.5, -1.0, 1.0, 0.0, -2.2], device=DEV, dtype=torch.float64)
    near(loss, want, torch.full((8,), 1e-4, device=DEV), "loss")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lengths,vocab,behind", [
    ([1, 1], 1, 0), ([3, 5], 65, 2), ([4, 0, 0, 7], 1000, 1), ([0, 0], 33, 4), ([20, 31, 17, 1, 9, 300], 513, 3),
    ([3, 2], 151_936, 1), ([700, 600], 130, 0)])
@pytest.mark.parametrize("before", [0, 2])
def test_preference_loss(scorer, lengths, vocab, behind, before, dtype):
    T, beta, smooth = 1.0, 0.1, 0.1 * (before > 0)
    start = np.concatenate([[before], before + np.cumsum(lengths)]).astype(np.int32)
    rows, pairs = int(start[-1]) + behind, len(lengths) // 2
    x, g = make_logits(rows, vocab, dtype, seed=rows + vocab, pad=vocab % 3, shift=rows % 4)
    token = ids_of(x, g, masked=0.3)
    r = torch.randn(2 * pairs, generator=g, device=DEV) * 5
    w = torch.rand(pairs, generator=g, device=DEV) + 0.5
    if pairs > 1:
        w[0] = 0.0
    loss, logprob, err = out(pairs), out(2 * pairs), records(pairs)
    full = torch.full((rows, vocab + 1), 5.0, dtype=x.dtype, device=DEV)
    d_start = torch.from_numpy(start).to(DEV)
    # rows outside the sequences are not looked at
    x = x.clone()
    x[:before] = math.nan
    x[int(start[-1]):] = math.nan
    token[:before] = vocab + 3
    scorer.preference_loss(x, token.int(), d_start, ref_logprob=r, weight=w, beta=beta, label_smoothing=smooth,
                           loss=loss, logprob=logprob, grad=full[:, :vocab], err=err, temperature=T)
    inside = slice(before, int(start[-1]))
    assert not read_errors(err).view(np.uint8).any()
    assert (full[:before] == 5.0).all() and (full[int(start[-1]):] == 5.0).all() and (full[:, vocab:] == 5.0).all()
    if inside.start == inside.stop:
        near(loss, torch.nn.functional.softplus(-beta * -(r[0::2] - r[1::2]).double()) * (1 - smooth)
             + smooth * torch.nn.functional.softplus(beta * -(r[0::2] - r[1::2]).double()),
             torch.full((pairs,), 1e-6, device=DEV), "loss")
        return
    xs, ts = x[inside], token[inside]
    want = ref.preference(xs, ts, (start - before).tolist(), beta, T, smooth, r, w)
    row_tol = 2 * ref.lse_tolerance(xs, T)
    seq_tol = torch.stack([row_tol[a - before:b - before].sum() for a, b in zip(start[:-1], start[1:])])
    near(logprob, want["logprob"], ref.scalar_tolerance(want["logprob"], seq_tol), "logprob")
    h_tol = beta * (seq_tol[0::2] + seq_tol[1::2])
    near(loss, want["loss"], ref.scalar_tolerance(want["loss"], h_tol), "loss")
    # the slope moves by at most beta h_tol / 4; that error goes with (delta - q)
    seq = torch.repeat_interleave(torch.arange(2 * pairs, device=DEV), torch.tensor(lengths, device=DEV))
    scale = want["slope"].abs()[seq // 2]
    slip = (beta * w.double() / T * h_tol)[seq // 2]
    q = torch.softmax(xs.double() / T, 1)
    one = torch.zeros_like(q)
    live = (ts >= 0) & (w[seq // 2] != 0)
    one[live, ts[live]] = 1.0
    slip = torch.where(live, slip, 0.0)
    bound = ref.grad_tolerance(want["grad"], scale[:, None], q, row_tol[:, None], x.dtype)
    bound = bound + slip[:, None] * (one - q).abs() + scale[:, None] * one * q * row_tol[:, None]
    near(full[inside, :vocab], want["grad"], bound, "grad")


# ---- values that a sum could lose ----

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 1200])
def test_extreme_rows(scorer, rows, dtype):
    """Masked chunks of every place, one large logit late or early, all far below 0, far apart, the type's lowest."""
    vocab = 9001
    x, g = make_logits(rows, vocab, dtype, seed=8)
    low = torch.finfo(x.dtype).min
    kinds = 8
    for r in range(rows):
        kind = r % kinds if rows > 2 else r
        if kind == 0:
            x[r, :4096] = -math.inf
        elif kind == 1:
            x[r, 8999] = 300.0
        elif kind == 2:
            x[r, 3] = 300.0
        elif kind == 3:
            x[r] = x[r] - 500.0
            x[r, :4096] = -math.inf
        elif kind == 4:
            x[r, 1:] = low
        elif kind == 5:
            x[r, 4096:] = low
        elif kind == 6:
            x[r] = x[r] * 1000.0
        else:
            x[r, :-1] = -math.inf
            x[r, -1] = -400.0
    token = x.float().argmax(1)
    lp, lse, ent = out(rows), out(rows), out(rows)
    err = records(rows)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, entropy=ent, err=err)
    want = ref.logprobs(x, token)
    tol = ref.lse_tolerance(x, 1.0)
    assert not read_errors(err).view(np.uint8).any()
    near(lse, want["lse"], ref.scalar_tolerance(want["lse"], tol), "lse")
    near(lp, want["logprob"], ref.scalar_tolerance(want["logprob"], 2 * tol), "logprob")
    near(ent, want["entropy"], ref.scalar_tolerance(want["entropy"], 4 * tol), "entropy")
    grad, loss = torch.full_like(x, 5.0), out(rows)
    one = torch.ones(rows, device=DEV)
    scorer.policy_loss(x, token.int(), lp, one, loss=loss, grad=grad)
    want = ref.policy(x, token, lp, one)
    near_grad(grad, want["grad"], one.double() * 1.1, x, 1.0, 2 * tol + ref.EPS32 * 60)
    assert (grad[torch.isinf(x)] == 0).all()


# ---- rows that are skipped, and rows that fail ----

@pytest.mark.parametrize("rows", [7, 1200])
def test_skipped_rows_are_not_read(scorer, rows):
    vocab = 2048
    x, g = make_logits(rows, vocab, "bf16", seed=2)
    token = ids_of(x, g)
    token[::2] = -1
    x[::2] = math.nan
    lp, lse, ent, err = out(rows), out(rows), out(rows), records(rows)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, entropy=ent, err=err)
    assert not read_errors(err).view(np.uint8).any()
    assert (lp[::2] == 0).all() and (lse[::2] == 0).all() and (ent[::2] == 0).all()
    assert torch.isfinite(lp).all() and (lp[1::2] < 0).all()
    for call in ("policy", "distill", "grad"):
        grad, loss = torch.full_like(x, 5.0), out(rows)
        w = torch.ones(rows, device=DEV)
        if call == "policy":
            scorer.policy_loss(x, token.int(), lp, w, loss=loss, grad=grad)
        elif call == "distill":
            w[::2] = 0.0
            ids = torch.arange(4, device=DEV).repeat(rows, 1)
            scorer.distill_loss(x, ids.int(), ids.float(), weight=w, loss=loss, grad=grad)
        else:
            scorer.token_logprobs_grad(x, token.int(), lse, grad=grad, grad_logprob=w)
            loss = torch.zeros(rows, device=DEV)
        assert (grad[::2] == 0).all() and torch.isfinite(grad).all() and (grad[1::2] != 0).any(1).all(), call
        assert (loss[::2] == 0).all() and torch.isfinite(loss).all(), call


@pytest.mark.parametrize("rows", [6, 1200])
def test_failed_rows_have_records(scorer, rows):
    vocab = 3001
    x, g = make_logits(rows, vocab, "f32", seed=4)
    token = ids_of(x, g)
    x[0, 2999] = math.inf
    x[0, 3000] = math.nan
    x[1, 5] = math.nan
    x[2] = -math.inf
    token[3] = vocab
    x[4] = torch.finfo(torch.float32).min  # out of range once scaled: weighs nothing
    lp, lse, ent, err = out(rows), out(rows), out(rows), records(rows)
    scorer.token_logprobs(x, token.int(), logprob=lp, lse=lse, entropy=ent, err=err)
    e = read_errors(err)
    nf = s.NONFINITE_OUTPUT
    assert e["status"][:6].tolist() == [nf, nf, nf, s.TOKEN_ID, nf, 0] and not e["status"][6:].any()
    assert e["position"][:5].tolist() == [0, 1, 2, 3, 4]
    assert [int(d) & 0xFFFFFFFF for d in e["detail"][:3]] == [2999, 5, 0]
    assert (int(e["needed"][3]), int(e["available"][3])) == (vocab, vocab)
    assert int(e["available"][0]) == 0x7F800000
    assert lp[:5].isnan().all() and lse[:5].isnan().all() and ent[:5].isnan().all() and torch.isfinite(lp[5:]).all()
    grad, loss, one = torch.full_like(x, 5.0), out(rows), torch.ones(rows, device=DEV)
    scorer.policy_loss(x, token.int(), torch.zeros(rows, device=DEV), one, loss=loss, grad=grad, err=err)
    assert (read_errors(err)["status"] == e["status"]).all()
    assert grad[:5].isnan().all() and loss[:5].isnan().all() and torch.isfinite(grad[5:]).all()
    grad.fill_(5.0)
    scorer.token_logprobs_grad(x, token.int(), lse, grad=grad, grad_logprob=one)
    assert grad[:5].isnan().all() and torch.isfinite(grad[5:]).all()
    ids, value = out(rows, 3, dtype=torch.int32, fill=9), out(rows, 3)
    scorer.top_logits(x, 3, token=ids, value=value, lse=lse, err=err)
    e = read_errors(err)
    assert e["status"][:6].tolist() == [nf, nf, nf, 0, nf, 0]
    assert (ids[[0, 1, 2, 4]] == -1).all() and value[[0, 1, 2, 4]].isnan().all() and (ids[5:] >= 0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_failed_distill_rows_have_records(scorer, tail):
    rows, vocab, k = 9, 700, 6
    x, g = make_logits(rows, vocab, "f32", seed=6)
    ids, logit, lse = teacher(x, g, k, 1.0, short=False)
    ids[0, 2] = vocab
    ids[1, 4] = ids[1, 1]
    logit[2, 3] = math.nan
    logit[3, 5] = math.inf
    x[4, ids[4, 0]] = math.nan
    x[5, 650] = math.inf
    lse[6] = math.inf
    x[7] = -math.inf
    loss, grad, err = out(rows), out(rows, vocab), records(rows)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse if tail else None, loss=loss, grad=grad, err=err)
    e = read_errors(err)
    want = [s.TOKEN_ID, s.TOKEN_ID, s.NONFINITE_INPUT, s.NONFINITE_INPUT, s.NONFINITE_OUTPUT, s.NONFINITE_OUTPUT,
            s.NONFINITE_INPUT if tail else 0, s.NONFINITE_OUTPUT, 0]
    assert e["status"].tolist() == want
    low = [int(d) & 0xFFFFFFFF for d in e["detail"]]
    first_nan = min(int(ids[4, 0]), vocab)
    assert low[:6] == [2, 1, 3, 5, first_nan, 650]
    bad = torch.tensor(want) != 0
    assert loss.cpu()[bad].isnan().all() and grad.cpu()[bad].isnan().all()
    assert torch.isfinite(loss.cpu()[~bad]).all() and torch.isfinite(grad.cpu()[~bad]).all()


def test_failed_pairs_have_records(scorer):
    vocab = 100
    start = torch.tensor([0, 3, 6, 9, 12, 15, 14, 20, 31], dtype=torch.int32, device=DEV)
    x, g = make_logits(30, vocab, "f32", seed=6)
    token = ids_of(x, g)
    x[4, 50] = math.nan
    token[7] = vocab + 1
    loss, logprob, grad, err = out(4), out(8), torch.full((30, vocab), 5.0, device=DEV), records(4)
    scorer.preference_loss(x, token.int(), start, beta=0.1, loss=loss, logprob=logprob, grad=grad, err=err)
    e = read_errors(err)
    assert e["status"].tolist() == [s.NONFINITE_OUTPUT, s.TOKEN_ID, s.CAPACITY, s.CAPACITY]
    assert e["position"].tolist() == [4, 7, 2, 3]
    assert (int(e["needed"][3]), int(e["available"][3])) == (30, 31)
    assert loss.isnan().all() and logprob.isnan().all()
    assert grad[:12].isnan().all() and (grad[12:] == 5.0).all()


@pytest.mark.parametrize("vocab", [2000, 2003])
@pytest.mark.parametrize("operator", ["policy", "distill", "preference"])
def test_outliers_cost_no_precision(scorer, operator, vocab):
    """Two outliers far above everything a thread has met before them hold a 32-bit row's mass.

    The factor of 2^(x c - shift) that each sum and gradient rounds to is near 1 for them if the shift follows:
    an element's gradient is then off, relatively, by 2 (2^-23 + 4 2^-24) from the sums (in q and in the slope),
    2^-23 from its own exponential, 5 2^-24 from the products, the gradient's rounding and a, and 2^-25 of what
    separates the two.  About a shift that stays 49 below, a alone may be off by 2^-19 / 2 ln 2 in each of the two."""
    rows, T = 400, 0.7
    x, g = make_logits(rows, vocab, "f32", seed=vocab)
    x.clamp_(max=10.0)
    each = torch.arange(rows, device=DEV)
    one, two = 1100 + each % 300, 1500 + each % 350
    x[each, one] = 26.0 + torch.rand(rows, generator=g, device=DEV)
    x[each, two] = x[each, one] - 0.5 * torch.rand(rows, generator=g, device=DEV)
    token, grad, loss = two, out(rows, vocab), out(rows)
    q = torch.softmax(x.double() / T, 1)
    lp = torch.log(q[each, token])
    if operator == "policy":
        old, adv = lp.float() + 0.05, torch.ones(rows, device=DEV)
        scorer.policy_loss(x, token.int(), old, adv, loss=loss, grad=grad, temperature=T, clip_low=0.2, clip_high=0.2)
        slope = -torch.exp(lp - old.double()) / T
    elif operator == "distill":
        scorer.distill_loss(x, token.int()[:, None], torch.zeros((rows, 1), device=DEV), loss=loss, grad=grad,
                            temperature=T)
        slope = torch.full_like(lp, -1.0 / T)
    else:
        start = torch.arange(rows + 1, dtype=torch.int32, device=DEV)
        scorer.preference_loss(x, token.int(), start, beta=0.1, loss=out(rows // 2), grad=grad, temperature=T)
        h = 0.1 * (lp[0::2] - lp[1::2])
        slope = torch.stack([-torch.sigmoid(-h), torch.sigmoid(-h)], 1).flatten() * 0.1 / T
    want = -slope * q[each, one]
    tol = (2 * 6 * 2.0 ** -24 + 2 * 2.0 ** -24 + 5 * 2.0 ** -24 + 2 * 2.0 ** -25) * want.abs()
    near(grad[each, one], want, tol, "gradient")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("rise", [12.0, 60.0, 400.0, 30_000.0])
def test_bad_logits_fail_under_later_larger_ones(scorer, dtype, bad, rise):
    """A thread that has met a NaN or an infinity reports it whatever its later chunks hold."""
    vocab, rows, at = 20_011, 70, 9
    x, g = make_logits(rows, vocab, dtype, seed=3)
    token = ids_of(x, g).int()
    x[1, at] = bad
    x[:, at + 1024::1024] = rise
    x[:, at + 5::2048] = rise + 1.0
    lp, ent, loss, grad, err = out(rows), out(rows), out(rows), torch.zeros_like(x), records(rows)
    ids, value = out(rows, 5, dtype=torch.int32, fill=0), out(rows, 5)

    def check():
        e = read_errors(err)
        assert e["status"][1] == s.NONFINITE_OUTPUT and int(e["detail"][1]) & 0xFFFFFFFF == at
        assert (e["status"] != 0).sum() == 1

    scorer.token_logprobs(x, token, logprob=lp, entropy=ent, err=err)
    check()
    scorer.top_logits(x, 5, token=ids, value=value, err=err)
    check()
    for n in (2, rows):
        few = records(n)
        scorer.policy_loss(x[:n], token[:n], torch.zeros_like(loss[:n]), torch.ones_like(loss[:n]), loss=loss[:n],
                           grad=grad[:n], err=few)
        assert read_errors(few)["status"][1] == s.NONFINITE_OUTPUT and grad[1].isnan().all()
    good = torch.arange(rows, device=DEV) != 1
    assert lp[1].isnan() and torch.isfinite(lp[good]).all() and torch.isfinite(ent[good]).all()


@pytest.mark.parametrize("more", [0, 40, 5000])
def test_pairs_that_share_rows_fail(scorer, more):
    """Offsets that fall back would give rows to two pairs: they are the last sequence's alone."""
    vocab, tail = 70, torch.arange(41, 41 + 2 * more)  # `more` pairs of one-row sequences behind the others
    start = torch.cat([torch.tensor([0, 2, 6, 6, 8, 20, 3, 5, 7, 21, 40]), tail]).to(torch.int32)
    pairs, rows = start.numel() // 2, int(start[-1]) + 2
    x, g = make_logits(rows, vocab, "f32", seed=60 + more)
    token = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    lp = torch.log_softmax(x.double(), 1).gather(1, token[:, None])[:, 0]

    def per_sequence(v):
        return torch.cat([v.new_zeros(1), v.cumsum(0)])[start.to(DEV).long()].diff()[6:]

    tol = ref.scalar_tolerance(per_sequence(lp), per_sequence(2 * ref.lse_tolerance(x, 1.0)))
    for _ in range(3):
        loss, logprob, grad, err = out(pairs), out(2 * pairs), torch.full((rows, vocab), 5.0, device=DEV), records(pairs)
        scorer.preference_loss(x, token.int(), start.to(DEV), beta=0.1, loss=loss, logprob=logprob, grad=grad, err=err)
        # the sequences: 0-1, 2-5 | none, 6-7 | 8-19, back to 3 | 3-4, 5-6 | 7-20, 21-39 | ...
        e = read_errors(err)
        want_bad = [True, True, True, False, False] + [False] * (pairs - 5)
        assert (e["status"] == s.CAPACITY).tolist() == want_bad and (e["status"] != 0).tolist() == want_bad
        bad = torch.tensor(want_bad)
        assert loss.cpu()[bad].isnan().all() and logprob.cpu().view(-1, 2)[bad].isnan().all()
        near(logprob[6:], per_sequence(lp), tol, "logprob")
        assert (grad[:3] == 5.0).all() and (grad[-2:] == 5.0).all()
        assert torch.isfinite(grad[3:rows - 2]).all() and (grad[3:rows - 2] != 5.0).all()


# ---- how calls are made ----

def all_calls(sc, x, token, g, stream=None):
    """Every operator bound on fixed buffers: (calls, outputs)."""
    rows, vocab = x.shape
    k = 5
    ids = torch.topk(x.float(), k, dim=1).indices.int()
    logit = torch.randn((rows, k), generator=g, device=DEV)
    half = rows // 2
    start = torch.tensor([0, half, rows], dtype=torch.int32, device=DEV)
    o = dict(lp=out(rows), lse=out(rows), ent=out(rows), loss=out(rows), loss2=out(rows), loss3=out(1),
             top=out(rows, k, dtype=torch.int32, fill=0), value=out(rows, k),
             **{f"grad{i}": torch.zeros_like(x) for i in range(4)})
    one = torch.ones(rows, device=DEV)
    old = torch.full((rows,), -3.0, device=DEV)
    kw = dict(stream=stream)
    calls = [
        sc.bind_token_logprobs(x, token, logprob=o["lp"], lse=o["lse"], entropy=o["ent"], **kw),
        sc.bind_token_logprobs_grad(x, token, o["lse"], grad=o["grad0"], grad_logprob=one, grad_entropy=one,
                                    entropy=o["ent"], **kw),
        sc.bind_top_logits(x, k, token=o["top"], value=o["value"], **kw),
        sc.bind_distill_loss(x, ids, logit, teacher_lse=torch.logsumexp(logit, 1) + 0.1, loss=o["loss"],
                             grad=o["grad1"], **kw),
        sc.bind_policy_loss(x, token, old, one, loss=o["loss2"], grad=o["grad2"], **kw),
        sc.bind_preference_loss(x, token, start, beta=0.1, loss=o["loss3"], grad=o["grad3"], **kw),
    ]
    return calls, o


@pytest.mark.parametrize("rows", [3, 600])
def test_captured_calls_replay(rows):
    """One graph of all operators, replayed on changing logits with eager work between, against eager calls."""
    vocab = 2011
    sc = RowScorer(0)
    sc.reserve(rows, vocab)
    x, g = make_logits(rows, vocab, "bf16", seed=1)
    x = x.contiguous()
    token = ids_of(x, g).int()
    hs = hip.Stream()
    calls, o = all_calls(sc, x, token, g, stream=hs)
    torch.cuda.synchronize()
    graph = hip.Graph(hs)
    graph.begin()
    for c in calls:
        c()
    graph.end()
    for step in range(4):
        fresh, _ = make_logits(rows, vocab, "bf16", seed=50 + step)
        x.copy_(fresh)
        for v in o.values():
            v.zero_()
        torch.cuda.synchronize()
        graph.launch()
        hs.synchronize()
        got = {k: v.clone() for k, v in o.items()}
        for v in o.values():
            v.zero_()
        torch.cuda.synchronize()
        for c in calls:
            c()
        hs.synchronize()
        for k, v in o.items():
            assert torch.equal(got[k], v), (step, k)
    graph.close()
    sc.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(2, 151_936), (5, 333), (1200, 700)])
def test_gradient_in_place_of_the_logits(scorer, rows, vocab, dtype):
    x, g = make_logits(rows, vocab, dtype, seed=1)
    x = x.contiguous()
    token = ids_of(x, g, masked=0.1).int()
    lp, lse = out(rows), out(rows)
    scorer.token_logprobs(x, token, logprob=lp, lse=lse)
    one = torch.ones(rows, device=DEV)
    ids = torch.topk(x.float(), 9, dim=1).indices.int()
    logit = torch.randn((rows, 9), generator=g, device=DEV)
    start = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=DEV)
    t_lse = torch.logsumexp(logit, 1) + 0.1
    for name in ("grad", "distill", "policy", "preference"):
        got = []
        for inplace in (False, True):
            y = x.clone()
            grad = y if inplace else torch.zeros_like(y)
            loss = out(rows)
            if name == "grad":
                scorer.token_logprobs_grad(y, token, lse, grad=grad, grad_logprob=one)
            elif name == "distill":
                scorer.distill_loss(y, ids, logit, teacher_lse=t_lse, loss=loss, grad=grad)
            elif name == "policy":
                scorer.policy_loss(y, token, lp - 0.1, one, loss=loss, grad=grad)
            else:
                scorer.preference_loss(y, token, start, beta=0.1, loss=loss, grad=grad)
            got.append((grad.clone(), torch.nan_to_num(loss)))
        assert torch.equal(got[0][0], got[1][0]), name
        assert torch.equal(got[0][1], got[1][1]), name


def test_two_contexts_on_two_streams():
    """Contexts are independent: the same calls on two streams at once give what each gives alone."""
    rows, vocab = 300, 5003
    scs = [RowScorer(0), RowScorer(0)]
    made = [make_logits(rows, vocab, "bf16", seed=9 + i) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    bound = []
    for sc, (x, g), st in zip(scs, made, streams):
        sc.reserve(rows, vocab)
        bound.append(all_calls(sc, x, ids_of(x, g).int(), g, stream=st))
    torch.cuda.synchronize()
    want = []
    for calls, o in bound:
        for c in calls:
            c()
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in o.items()})
    for _, o in bound:
        for v in o.values():
            v.zero_()
    torch.cuda.synchronize()
    for a, b in zip(bound[0][0], bound[1][0]):
        a()
        b()
    torch.cuda.synchronize()
    for (_, o), w in zip(bound, want):
        for k in o:
            assert torch.equal(o[k], w[k]), k
    for sc in scs:
        sc.close()


def test_device_arrays_without_torch(scorer):
    """The framework's own buffers: binary32 words, and 16-bit words with a named type."""
    rng = np.random.default_rng(3)
    x = rng.normal(0, 2, (4, 600)).astype(np.float32)
    token = np.array([1, 599, 0xFFFFFFFF, 7], np.uint32)
    dev = hip.DeviceArray.from_numpy
    lp = hip.DeviceArray(4, np.float32)
    scorer.token_logprobs(dev(x.view(np.uint32)), dev(token), logprob=lp)
    want = ref.logprobs(torch.from_numpy(x), torch.tensor([1, 599, -1, 7]))["logprob"]
    assert np.abs(lp.numpy() - want.numpy()).max() < 1e-5
    half = (x.view(np.uint32) >> 16).astype(np.uint16)  # cut to bfloat16
    cut = (half.astype(np.uint32) << 16).view(np.float32)
    scorer.token_logprobs(dev(half), dev(token), logprob=lp, dtype="bf16")
    want = ref.logprobs(torch.from_numpy(cut), torch.tensor([1, 599, -1, 7]))["logprob"]
    assert np.abs(lp.numpy() - want.numpy()).max() < 1e-5
    with pytest.raises(ValueError):
        scorer.token_logprobs(dev(half), dev(token), logprob=lp)


def test_results_repeat(scorer):
    x, g = make_logits(64, 20_011, "f32", seed=5)
    token = ids_of(x, g).int()
    calls, o = all_calls(scorer, x, token, g)
    runs = []
    for _ in range(3):
        for c in calls:
            c()
        torch.cuda.synchronize()
        runs.append({k: v.clone() for k, v in o.items()})
    for k in o:
        assert torch.equal(runs[0][k], runs[1][k]) and torch.equal(runs[0][k], runs[2][k]), k


def test_teacher_to_student_and_rollout_to_policy(scorer):
    """The operators as they are used together: a teacher's record distilled; a decode step's tokens scored, then
    trained on: both losses fall along their gradients."""
    rows, vocab, k, T = 12, s.VOCAB, 20, 2.0
    teach, g = make_logits(rows, vocab, "bf16", seed=21)
    x = (teach.float() + torch.randn(teach.shape, generator=g, device=DEV)).contiguous()
    ids, value, lse = out(rows, k, dtype=torch.int32, fill=0), out(rows, k), out(rows)
    scorer.top_logits(teach, k, token=ids, value=value, lse=lse, temperature=T)
    loss, grad, after = out(rows), torch.empty_like(x), out(rows)
    scorer.distill_loss(x, ids, value, teacher_lse=lse, loss=loss, grad=grad, temperature=T)
    scorer.distill_loss(x - 0.1 * grad, ids, value, teacher_lse=lse, loss=after, temperature=T)
    assert (loss > 0).all() and (after < loss).all()
    # the directional derivative is the gradient's square
    slope = (loss - after).double() / 0.1
    square = grad.double().square().sum(1)
    assert ((slope - square).abs() <= 0.1 * square + 1e-4).all()

    batch = s.DecodeBatch([[1, 2, 3]] * rows, list(range(1, rows + 1)), [8] * rows, device=0)
    tokens = batch.step(x)
    assert (tokens != s.NO_TOKEN).all()
    token = torch.from_numpy(tokens.view(np.int32)).to(DEV)
    behaviour = out(rows)
    scorer.token_logprobs(x, token, logprob=behaviour, temperature=0.7)
    loss, kl, lp = out(rows), out(rows), out(rows)
    adv = torch.linspace(-1, 1, rows, device=DEV)
    scorer.policy_loss(x, token, behaviour, adv, ref_logprob=behaviour, kl_coef=0.1, loss=loss, kl=kl, logprob=lp,
                       grad=grad, temperature=0.7)
    # on policy: the ratio is 1 up to the behaviour's own rounding (its half step), the KL its square
    half = ref.EPS32 * behaviour.double().abs() + 1e-12
    near(loss, -adv.double(), 1.1 * half + ref.EPS32 * adv.double().abs(), "loss")
    assert (kl.abs() <= 1e-12).all() and torch.equal(lp, behaviour)
    batch.close()


def test_decode_steps_return_log_probabilities(scorer):
    """A decode batch's own log-probabilities: of the tokens it drew, 0 for rows that have ended."""
    rows, T = 5, 0.7
    batch = s.DecodeBatch([[1, 2, 3]] * rows, list(range(7, 7 + rows)), [1, 4, 4, 2, 4], device=0)
    plain = s.DecodeBatch([[1, 2, 3]] * rows, list(range(7, 7 + rows)), [1, 4, 4, 2, 4], device=0)
    for step in range(4):
        x, g = make_logits(rows, s.VOCAB, "f32", seed=60 + step)
        lp = out(rows)
        tokens = batch.step(x, logprobs=lp, logprob_temperature=T)
        assert (tokens == plain.step(x)).all()
        token = torch.from_numpy(tokens.view(np.int32)).to(DEV).long()
        want = ref.logprobs(x, token, T)["logprob"]
        near(lp, want, ref.scalar_tolerance(want, 2 * ref.lse_tolerance(x, T)), "logprob")
        assert ((token >= 0) == (lp != 0)).all()
    assert (tokens[[0, 3]] == s.NO_TOKEN).all() and batch.active() == plain.active()
    before = [st.state() for st in batch.sampling_states()]
    for bad in (dict(logprobs=torch.zeros(rows)), dict(logprobs=out(rows - 1)), dict(logprobs=out(rows, dtype=torch.float64)),
                dict(logprobs=out(rows), logprob_temperature=0.0)):
        with pytest.raises(ValueError):
            batch.step(x, **bad)
    assert [st.state() for st in batch.sampling_states()] == before
    batch.close()
    plain.close()


def test_a_closed_scorer_refuses_its_calls():
    sc = RowScorer(0)
    x, g = make_logits(2, 50, "f32")
    call = sc.bind_token_logprobs(x, ids_of(x, g).int(), logprob=out(2))
    call()
    torch.cuda.synchronize()
    sc.close()
    with pytest.raises(ValueError):
        call()
    with pytest.raises(ValueError):
        sc.token_logprobs(x, ids_of(x, g).int(), logprob=out(2))


def test_logits_just_past_the_range_fail_wherever_they_stand(scorer):
    """y / ln 2 out of binary32's range, in the first chunk of a thread and in a later one."""
    vocab = 40_000
    for at in (3, vocab - 5):
        for rows in (2, 1100):
            x, g = make_logits(rows, vocab, "f32", seed=1)
            x[1, at] = 2.2e38  # x log2(e) = 3.17e38
            lp, loss, grad, err = out(rows), out(rows), torch.full_like(x, 5.0), records(rows)
            token = ids_of(x, g).int()
            scorer.token_logprobs(x, token, logprob=lp, err=err)
            e = read_errors(err)
            assert e["status"][1] == s.NONFINITE_OUTPUT and int(e["detail"][1]) & 0xFFFFFFFF == at
            one = torch.ones(rows, device=DEV)
            scorer.policy_loss(x, token, one, one, loss=loss, grad=grad, err=err)
            e = read_errors(err)
            assert e["status"][1] == s.NONFINITE_OUTPUT and int(e["detail"][1]) & 0xFFFFFFFF == at
            assert lp[1].isnan() and loss[1].isnan() and grad[1].isnan().all() and torch.isfinite(grad[0]).all()
            x[1, at] = -2.2e38  # below the range: weighs nothing
            scorer.token_logprobs(x, token, logprob=lp, err=err)
            assert not read_errors(err)["status"].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,k,tail", [(70, 9001, 60, True), (70, 170_001, 90, True), (70, 170_001, 90, False),
                                               (600, 45_001, 128, True), (300, 25_003, 30, True), (2, 600_001, 100, True)])
def test_lists_that_reach_every_part_of_a_row(scorer, dtype, rows, vocab, k, tail):
    """Listed ids in the chunks that are held, kept in LDS and read again, neighbours in one chunk, the row's last."""
    x, g = make_logits(rows, vocab, dtype, seed=vocab + k)
    ids = torch.linspace(0, vocab - 1, k, device=DEV).long().repeat(rows, 1)
    ids[:, 1], ids[:, 2], ids[:, k - 2] = 1, 2, vocab - 2
    logit = torch.randn((rows, k), generator=g, device=DEV)
    lse = (torch.logsumexp(logit.double(), 1) + 0.2).float() if tail else None
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    loss, grad = out(rows), torch.full_like(x, 5.0)
    scorer.distill_loss(x, ids.int(), logit, teacher_lse=lse, weight=w, loss=loss, grad=grad)
    tol = 2 * ref.lse_tolerance(x, 1.0)
    for lo in range(0, rows, 100):  # in 64 bits by parts
        r = slice(lo, lo + 100)
        part = None if lse is None else lse[r]
        want = ref.distill(x[r], ids[r], logit[r], 1.0, part, w[r])
        near(loss[r], want["loss"], ref.scalar_tolerance(want["loss"], tol[r]), "loss")
        near_grad(grad[r], want["grad"], distill_scale(x[r], ids[r], logit[r], 1.0, part, w[r]), x[r], 1.0, tol[r])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab", [(64, 155_650), (64, 33), (1030, 5003), (70, 80_003)])
def test_policy_tokens_in_every_part_of_a_row(scorer, dtype, rows, vocab):
    x, g = make_logits(rows, vocab, dtype, seed=vocab)
    token = torch.linspace(0, vocab - 1, rows, device=DEV).long()
    lp = ref.logprobs(x, token)["logprob"].float()
    adv = torch.ones(rows, device=DEV)
    loss, grad = out(rows), torch.full_like(x, 5.0)
    scorer.policy_loss(x, token.int(), lp, adv, loss=loss, grad=grad)
    want = ref.policy(x, token, lp, adv)
    tol = 2 * ref.lse_tolerance(x, 1.0) + ref.EPS32 * lp.double().abs()
    q = torch.softmax(x.double(), 1)
    one = torch.zeros_like(q).scatter_(1, token[:, None], 1.0)
    bound = ref.grad_tolerance(want["grad"], adv[:, None].double() * 1.1, q, tol[:, None], x.dtype)
    bound = bound + tol[:, None] * (one - q).abs() + one * q * tol[:, None]
    near(grad, want["grad"], bound, "grad")
