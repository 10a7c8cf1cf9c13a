"""The scores and losses of logits rows in 64 bits (torch), and how far 32-bit ones may be off.

Each function takes logits [rows, vocab] of any type and returns 64-bit outputs.  `token` is int64 with -1
for a row without one.
"""
import math

import torch

EPS32 = 2.0 ** -24  # half a step of binary32, relative


def _stats(x, T):
    y = x.double() / T
    lse = torch.logsumexp(y, 1)
    return y, lse, torch.exp(y - lse[:, None])


def _onehot(x, token):
    one = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    live = token >= 0
    one[live, token[live]] = 1.0
    return one


def logprobs(x, token, T=1.0):
    y, lse, q = _stats(x, T)
    live = token >= 0
    at = token.clamp(min=0)[:, None]
    logq = y - lse[:, None]
    entropy = -torch.where(q > 0, q * logq, 0.0).sum(1)
    zero = torch.zeros_like(lse)
    return dict(logprob=torch.where(live, logq.gather(1, at)[:, 0], zero), lse=torch.where(live, lse, zero),
                entropy=torch.where(live, entropy, zero))


def logprobs_grad(x, token, g, ge, T=1.0):
    y, lse, q = _stats(x, T)
    live = (token >= 0)[:, None]
    logq = torch.where(q > 0, y - lse[:, None], torch.zeros_like(y))
    entropy = -(q * logq).sum(1)
    grad = g[:, None].double() * (_onehot(x, token) - q) - ge[:, None].double() * q * (logq + entropy[:, None])
    return torch.where(live, grad / T, 0.0)


def top(x, k):
    """Ids and values of the k largest of each row, the lowest id first among equal ones."""
    order = torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True)
    return order.indices[:, :k], order.values[:, :k]


def distill(x, ids, logits, T=1.0, lse=None, weight=None):
    y, norm, q = _stats(x, T)
    rows, k = ids.shape
    valid = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(valid, logits.double() / T, -math.inf)
    any_ = (t > -math.inf).any(1)
    base = lse.double() if lse is not None else torch.where(any_, torch.logsumexp(t, 1), 0.0)
    p = torch.where(any_[:, None], torch.exp(t - base[:, None]), 0.0)
    logq = (y - norm[:, None]).gather(1, at)
    loss = torch.where(p > 0, p * (torch.log(p) - logq), 0.0).sum(1)
    target = torch.zeros_like(y).scatter_add_(1, at, torch.where(valid, p, 0.0))
    off = torch.zeros_like(y).scatter_add_(1, at, valid.double()) == 0
    mass = p.sum(1)
    if lse is not None:
        left = torch.where(any_, (1.0 - mass).clamp(min=0.0), 0.0)
        rest = torch.where(off, q, 0.0).sum(1)
        left = torch.where(rest > 0, left, 0.0)
        loss = loss + torch.where(left > 0, left * (torch.log(left) - torch.log(rest)), 0.0)
        target = target + torch.where(off, q * torch.where(rest > 0, left / rest, 0.0)[:, None], 0.0)
        mass = mass + left
    w = torch.ones(rows, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    on = w != 0.0
    grad = torch.where(on[:, None], (q * mass[:, None] - target) * (w / T)[:, None], 0.0)
    return dict(loss=torch.where(on, loss, 0.0), lse=torch.where(on, norm, 0.0), grad=grad)


def policy(x, token, old, adv, T=1.0, ref=None, weight=None, low=0.2, high=0.2, kl_coef=0.0):
    y, lse, q = _stats(x, T)
    live = token >= 0
    if weight is not None:
        live = live & (weight != 0)
    lp = (y - lse[:, None]).gather(1, token.clamp(min=0)[:, None])[:, 0]
    ratio, adv = torch.exp(lp - old.double()), adv.double()
    a, b = ratio * adv, ratio.clamp(1.0 - low, 1.0 + high) * adv
    loss, slope = -torch.minimum(a, b), torch.where(a <= b, -a, 0.0)
    kl = torch.zeros_like(lp)
    if ref is not None:
        gap = ref.double() - lp
        kl = torch.expm1(gap) - gap
        loss, slope = loss + kl_coef * kl, slope - kl_coef * torch.expm1(gap)
    w = torch.ones_like(lp) if weight is None else weight.double()
    c = torch.where(live, slope * w / T, 0.0)
    grad = torch.where(live[:, None], c[:, None] * (_onehot(x, token) - q), 0.0)
    return dict(loss=torch.where(live, loss, 0.0), logprob=torch.where(live, lp, 0.0),
                kl=torch.where(live, kl, 0.0), grad=grad, slope=c)


def preference(x, token, start, beta, T=1.0, smooth=0.0, ref=None, weight=None):
    """grad is NaN in the rows outside the sequences, which a call leaves alone."""
    y, lse, q = _stats(x, T)
    pairs = (len(start) - 1) // 2
    lp = torch.where(token >= 0, (y - lse[:, None]).gather(1, token.clamp(min=0)[:, None])[:, 0], 0.0)
    sums = torch.stack([lp[a:b].sum() for a, b in zip(start[:-1], start[1:])])
    r = torch.zeros_like(sums) if ref is None else ref.double()
    h = beta * ((sums - r)[0::2] - (sums - r)[1::2])
    sp = torch.nn.functional.softplus
    loss = (1.0 - smooth) * sp(-h) + smooth * sp(h)
    w = torch.ones_like(h) if weight is None else weight.double()
    slope = (torch.sigmoid(h) - (1.0 - smooth)) * beta * w / T
    grad = torch.full(y.shape, math.nan, dtype=torch.float64, device=x.device)
    one = _onehot(x, token)
    for s in range(2 * pairs):
        a, b = start[s], start[s + 1]
        c = slope[s // 2] * (1.0 if s % 2 == 0 else -1.0)
        on = (token[a:b] >= 0)[:, None] & (w[s // 2] != 0)
        grad[a:b] = torch.where(on, c * (one[a:b] - q[a:b]), 0.0)
    on = w != 0
    return dict(loss=torch.where(on, loss, 0.0), logprob=torch.where(on.repeat_interleave(2), sums, 0.0), grad=grad,
                slope=slope)


# ---- how far off ----

def lse_tolerance(x, T, live=None):
    """Bound of a row's error of lse (and of ln q), absolute, before the output's own rounding.

    With e = 2^-24 and Y the row's largest |y| of a logit that can weigh (y within 100 of the largest):
    c = log2(e) / T rounded once: e Y; a = fma(x, c, -shift) rounded once, |a| <= 2 Y / ln 2: 2 e Y; a weight's
    exp2: 2 e; the tree of a chunk's eight: 3 e; a thread's sum over its chunks: at most 96 e (a thread takes at most
    96 chunks in these tests' sizes); the rescale to the wave's shift: 3 e.  Everything above that is summed in 64
    bits.
    """
    y = x.double() / T
    top = y.amax(1, keepdim=True)
    big = torch.where((y > top - 100.0) & torch.isfinite(y), y.abs(), 0.0).amax(1)
    return EPS32 * (3.0 * big + 104.0)


def scalar_tolerance(value, tol):
    """An output rounded to binary32 after an error of tol."""
    return tol + EPS32 * value.abs() + 1e-37


def grad_tolerance(grad, scale, q, tol, dtype):
    """Bound of a gradient element's error: 2^a (alpha + beta a) has the relative errors of 2^a (as ln q above,
    twice: its own and the shift's) and of the factors (4 roundings), all within 2 tol of `scale` q; then it is
    rounded to the type, by half a step, or half the smallest subnormal step."""
    info = torch.finfo(dtype)
    half = info.eps / 2 if dtype != torch.float32 else EPS32
    tiny = float(info.tiny) * info.eps
    return half * grad.abs() + scale * q * (2.0 * tol) * (1.0 + half) + tiny + 1e-37 * scale
