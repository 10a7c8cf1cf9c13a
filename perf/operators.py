"""The logits-row scores and losses' timed cases: what a rollout, a teacher and a trainer ask of rows of logits.

A case is one call (or a forward and its gradient) over `rows` rows of a `vocab`-token vocabulary:

    logprobs    RowScorer.token_logprobs: log-probability of each row's token, log-sum-exp and entropy;
                with "grad" also RowScorer.token_logprobs_grad, as an external loss' backward asks for it.
    top         RowScorer.top_logits: a teacher's k largest logits of each row, and its log-sum-exp.
    distill     RowScorer.distill_loss: divergence from a teacher's top logits, and its gradient.
    policy      RowScorer.policy_loss: clipped policy loss with a KL term, and its gradient.
    preference  RowScorer.preference_loss: paired log ratios of chosen and rejected sequences, and the gradient.

Logits are N(0, 2.5^2) with five boosted ids, the distribution of promptboot_amd.workloads; tokens are drawn from
them.  Rows that a batch's mask leaves out carry the id NO_TOKEN.  Everything is made on the GPU from the seed.
"""
import math

import torch

own = False

V = 151_936  # the model's vocabulary
NO_TOKEN = -1  # 0xffffffff as the int32 that torch holds
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST = 2 * 2 * 4096 * V  # bytes of logits and gradient in the largest case
TILE = 256  # rows that are made, or worked out in 64 bits, together


def listed():
    return [
        # serving: the log-probability of one conversation's token, from the head's 32-bit row
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=V, dtype="f32", T=1.0, grad=False, masked=0.0, pad=0),
        # a rollout scored with a vocabulary whose rows start at any element, sampler's temperature
        dict(name="logprobs_70_odd", kind="logprobs", rows=70, vocab=50_257, dtype="f16", T=0.7, grad=False,
             masked=0.1, pad=0),
        # a training microbatch, entropy bonus: forward and gradient
        dict(name="logprobs_grad_1000", kind="logprobs", rows=1000, vocab=V, dtype="bf16", T=1.0, grad=True,
             masked=0.25, pad=0),
        # a teacher's record, few rows of 32 bits
        dict(name="top_33", kind="top", rows=33, vocab=V, dtype="f32", T=1.0, k=64),
        # a teacher's record of a whole batch; bf16 logits tie all the time
        dict(name="top_2048", kind="top", rows=2048, vocab=V, dtype="bf16", T=2.0, k=20),
        # distillation of a short answer, 32-bit logits, the teacher's remaining mass as one bucket
        dict(name="distill_12_tail", kind="distill", rows=12, vocab=V, dtype="f32", T=2.0, k=20, tail=True, masked=0.0,
             pad=0),
        # an ordinary microbatch in padded rows of another vocabulary
        dict(name="distill_700", kind="distill", rows=700, vocab=100_003, dtype="f16", T=1.0, k=100, tail=True,
             masked=0.2, pad=5),
        # the largest: a full batch of rows, bf16
        dict(name="distill_4096", kind="distill", rows=4096, vocab=V, dtype="bf16", T=2.0, k=64, tail=False,
             masked=0.0, pad=0),
        # a few rows of a policy step, latency of a fused forward and gradient
        dict(name="policy_5", kind="policy", rows=5, vocab=32_000, dtype="bf16", T=1.0, ref=False, masked=0.0, pad=0),
        # a policy step's microbatch, prompt rows masked
        dict(name="policy_2500", kind="policy", rows=2500, vocab=V, dtype="bf16", T=1.0, ref=True, masked=0.3, pad=0),
        # two pairs of short answers, 32-bit logits
        dict(name="preference_2", kind="preference", pairs=2, longest=60, vocab=V, dtype="f32", T=1.0, smooth=0.0,
             masked=0.4, pad=0),
        # a microbatch of pairs, ragged lengths, prompts masked, rows behind the last sequence
        dict(name="preference_8", kind="preference", pairs=8, longest=160, vocab=V, dtype="bf16", T=1.0, smooth=0.1,
             masked=0.4, pad=0),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["logprobs", "top", "distill", "policy", "preference"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    vocab = rng.choice([V, _log_uniform(rng, 1_000, 200_000)])
    case = dict(kind=kind, vocab=vocab, dtype=dtype, T=rng.choice([1.0, 1.0, 0.7, 2.0]))
    size = 4 if dtype == "f32" else 2
    fit = MOST // (2 * size * (vocab + 8))  # a drawn case moves no more than the largest listed one
    rows = _log_uniform(rng, 1, min(4096, fit))
    if kind == "top":
        return dict(case, rows=min(rows, 2048), k=_log_uniform(rng, 1, 128))
    case.update(masked=rng.choice([0.0, 0.1, 0.3]), pad=rng.choice([0, 0, 1, 8]))
    if kind == "logprobs":
        return dict(case, rows=rows, grad=rng.random() < 0.5)
    if kind == "distill":
        return dict(case, rows=rows, k=_log_uniform(rng, 1, 128), tail=rng.random() < 0.5)
    if kind == "policy":
        return dict(case, rows=rows, ref=rng.random() < 0.5)
    pairs = _log_uniform(rng, 1, 12)
    # the gradient reads a pair's rows again: half the rows, for the same traffic at most
    return dict(case, pairs=pairs, longest=max(1, min(400, rows // (4 * pairs))), smooth=rng.choice([0.0, 0.1]))


# ---- inputs, on the GPU, from the seed alone ----


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _integers(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _make_rows(case, rows, g):
    """Logits [rows, vocab] in rows of vocab + pad elements, and a token drawn from each."""
    vocab, dtype = case["vocab"], TYPES[case["dtype"]]
    full = torch.zeros((rows, vocab + case.get("pad", 0)), dtype=dtype, device="cuda")
    token = torch.empty(rows, dtype=torch.int32, device="cuda")
    for lo in range(0, rows, TILE):
        n = min(TILE, rows - lo)
        x = _randn(g, n, vocab).mul_(2.5)
        x.scatter_add_(1, _integers(g, 0, vocab, n, 5), _rand(g, n, 5) * 7.0 + 8.0)
        full[lo:lo + n, :vocab] = x
        y = full[lo:lo + n, :vocab].float() / case["T"]
        noise = -torch.log(-torch.log(_rand(g, n, vocab).clamp_(1e-20, 1.0 - 1e-7)))
        token[lo:lo + n] = (y + noise).argmax(1).int()
    return full[:, :vocab], token


def _mask(case, token, g):
    return torch.where(_rand(g, token.numel()) < case["masked"], NO_TOKEN, token)


def _logprob_of(logits, token, T):
    """The tokens' log-probabilities, for inputs that an earlier pass of a policy or a reference left."""
    out = torch.zeros(token.numel(), device="cuda")
    for lo in range(0, token.numel(), TILE):
        y = logits[lo:lo + TILE].float() / T
        t = token[lo:lo + TILE].long().clamp(min=0)
        out[lo:lo + TILE] = y.gather(1, t[:, None])[:, 0] - torch.logsumexp(y, 1)
    return out


def _lengths(case, g):
    """Row offsets of 2 x pairs sequences, and the rows of the buffer: three more than the sequences hold."""
    n = _integers(g, max(1, case["longest"] // 3), case["longest"] + 1, 2 * case["pairs"])
    start = torch.zeros(2 * case["pairs"] + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(n, 0)
    return start, 2 * case["pairs"] * case["longest"] + 3


CLIP_LOW, CLIP_HIGH, KL, BETA = 0.2, 0.28, 0.05, 0.1


def _scale(case):
    """What the rows' gradients are multiplied by: f16 training scales its loss, or the gradient underflows."""
    return 4096.0 if case["dtype"] == "f16" else 1.0


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, T = case["kind"], case["T"]
    d = {}
    if kind == "preference":
        d["start"], rows = _lengths(case, g)
    else:
        rows = case["rows"]
    d["logits"], token = _make_rows(case, rows, g)
    if kind == "top":
        return d
    if kind == "distill":
        # the teacher's logits: the student's at ids near its own top, moved
        k, vocab = case["k"], case["vocab"]
        ids = torch.empty((rows, k), dtype=torch.int32, device="cuda")
        for lo in range(0, rows, TILE):
            x = d["logits"][lo:lo + TILE].float()
            ids[lo:lo + TILE] = torch.topk(x + _rand(g, *x.shape), k, dim=1).indices.int()
        d["teacher_logit"] = d["logits"].gather(1, ids.long()).float() + _randn(g, rows, k)
        top = torch.logsumexp(d["teacher_logit"] / T, 1)
        if case["tail"]:  # 2 to 30 % of the teacher's mass is off its record
            d["teacher_lse"] = top - torch.log1p(-(_rand(g, rows) * 0.28 + 0.02))
        short = torch.arange(k, device="cuda")[None, :] >= _integers(g, (k + 1) // 2, k + 1, rows, 1)
        d["teacher_id"] = torch.where(short & (_rand(g, rows, 1) < 0.1), NO_TOKEN, ids)  # some records are short
        d["weight"] = torch.where(_rand(g, rows) < case["masked"], 0.0, _scale(case) / rows)
        return d
    d["token"] = _mask(case, token, g)
    if kind == "logprobs":
        if case["grad"]:
            d["grad_logprob"] = _randn(g, rows) * (_scale(case) / rows)
            d["grad_entropy"] = _rand(g, rows) * (-0.01 * _scale(case) / rows)
        return d
    if kind == "policy":
        lp = _logprob_of(d["logits"], token, T)
        old = lp + _randn(g, rows) * 0.15
        # a ratio within rounding of a clip bound has one gradient or none, by its last bit: keep clear of them
        for bound in (1.0 - CLIP_LOW, 1.0 + CLIP_HIGH):
            off = torch.exp(lp - old) - bound
            old = torch.where(off.abs() < 1e-3, old + 0.01, old)
        d["old"], d["advantage"] = old, _randn(g, rows)
        d["weight"] = torch.full((rows,), _scale(case) / rows, device="cuda")
        if case["ref"]:
            d["ref"] = lp + _randn(g, rows) * 0.3
        return d
    lp = torch.where(d["token"] >= 0, _logprob_of(d["logits"], token, T), 0.0).double().cumsum(0)
    ends = d["start"].long() - 1
    sums = torch.where(ends >= 0, lp[ends.clamp(min=0)], 0.0)
    d["ref"] = (sums[1:] - sums[:-1]).float() + _randn(g, 2 * case["pairs"]) * 4.0
    d["weight"] = torch.full((case["pairs"],), _scale(case) / case["pairs"], device="cuda")
    return d


def _zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    d = _inputs(case, seed)
    st = dict(case=case, d=d)
    if not own:
        return st
    from promptboot_amd.scores import RowScorer

    kind, T = case["kind"], case["T"]
    x = d["logits"]
    rows, vocab = x.shape
    sc = RowScorer(0)
    sc.reserve(rows, vocab)
    out, calls = {}, []
    if kind != "top" and (kind != "logprobs" or case["grad"]):
        out["grad"] = _zeros(rows, vocab, dtype=x.dtype)
    if kind == "logprobs":
        out.update(logprob=_zeros(rows), lse=_zeros(rows), entropy=_zeros(rows))
        calls.append(sc.bind_token_logprobs(x, d["token"], logprob=out["logprob"], lse=out["lse"],
                                            entropy=out["entropy"], temperature=T))
        if case["grad"]:
            calls.append(sc.bind_token_logprobs_grad(
                x, d["token"], out["lse"], grad=out["grad"], grad_logprob=d["grad_logprob"],
                grad_entropy=d["grad_entropy"], entropy=out["entropy"], temperature=T))
    elif kind == "top":
        out.update(id=_zeros(rows, case["k"], dtype=torch.int32), value=_zeros(rows, case["k"]), lse=_zeros(rows))
        calls.append(sc.bind_top_logits(x, case["k"], token=out["id"], value=out["value"], lse=out["lse"],
                                        temperature=T))
    elif kind == "distill":
        out.update(loss=_zeros(rows))
        calls.append(sc.bind_distill_loss(x, d["teacher_id"], d["teacher_logit"], teacher_lse=d.get("teacher_lse"),
                                          weight=d["weight"], loss=out["loss"], grad=out["grad"], temperature=T))
    elif kind == "policy":
        out.update(loss=_zeros(rows), logprob=_zeros(rows), kl=_zeros(rows))
        calls.append(sc.bind_policy_loss(
            x, d["token"], d["old"], d["advantage"], ref_logprob=d.get("ref"), weight=d["weight"],
            clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL if case["ref"] else 0.0, loss=out["loss"],
            logprob=out["logprob"], kl=out["kl"], grad=out["grad"], temperature=T))
    else:
        out.update(loss=_zeros(case["pairs"]), logprob=_zeros(2 * case["pairs"]))
        calls.append(sc.bind_preference_loss(
            x, d["token"], d["start"], ref_logprob=d["ref"], weight=d["weight"], beta=BETA,
            label_smoothing=case["smooth"], loss=out["loss"], logprob=out["logprob"], grad=out["grad"],
            temperature=T))
    return dict(st, scorer=sc, calls=calls, out=out)


def run(state):
    if not own:
        return _PLAIN[state["case"]["kind"]](state["case"], state["d"])
    for call in state["calls"]:
        call()
    return state["out"]


# ---- the plain form ----


def _softmax(x, T):
    """Scaled logits, their softmax and its log-sum-exp, in 32 bits."""
    y = x.float() / T
    top = y.amax(1, keepdim=True)
    e = torch.exp(y - top)
    s = e.sum(1, keepdim=True)
    return y, e / s, top[:, 0] + torch.log(s[:, 0])


def _plain_logprobs(case, d):
    y, q, lse = _softmax(d["logits"], case["T"])
    live = d["token"] >= 0
    t = d["token"].long().clamp(min=0)[:, None]
    entropy = lse - (q * y).sum(1)
    out = dict(logprob=torch.where(live, y.gather(1, t)[:, 0] - lse, 0.0), lse=torch.where(live, lse, 0.0),
               entropy=torch.where(live, entropy, 0.0))
    if case["grad"]:
        a = torch.where(live, d["grad_logprob"], 0.0)[:, None]
        b = torch.where(live, d["grad_entropy"], 0.0)[:, None]
        grad = -q * (a + b * (y - lse[:, None] + entropy[:, None]))
        grad.scatter_add_(1, t, a)
        out["grad"] = (grad / case["T"]).to(d["logits"].dtype)
    return out


def _plain_top(case, d):
    x = d["logits"].float() + 0.0  # -0 counts as 0
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)  # as whole numbers, in the values' order
    ids = torch.arange(x.shape[1], device="cuda")
    key = order * (1 << 24) - ids  # the lowest id of equal values first
    at = torch.topk(key, case["k"], dim=1).indices
    y = x / case["T"]
    top = y.amax(1, keepdim=True)
    return dict(id=at.int(), value=x.gather(1, at), lse=top[:, 0] + torch.log(torch.exp(y - top).sum(1)))


def _plain_distill(case, d):
    T = case["T"]
    y, q, lse = _softmax(d["logits"], T)
    live = d["teacher_id"] >= 0
    on = d["weight"] != 0.0
    at = d["teacher_id"].long().clamp(min=0)
    t = torch.where(live, d["teacher_logit"] / T, -math.inf)
    if case["tail"]:
        p = torch.exp(t - d["teacher_lse"][:, None])
    else:
        e = torch.exp(t - t.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    logq = y.gather(1, at) - lse[:, None]
    loss = torch.where(p > 0.0, p * (torch.log(p) - logq), 0.0).sum(1)
    grad = q.clone()
    if case["tail"]:
        rest = (1.0 - p.sum(1)).clamp(min=0.0)
        off = torch.ones_like(q)
        off.scatter_add_(1, at, torch.where(live, -1.0, 0.0))  # 1 off the teacher's ids, 0 on them
        mass = (q * off).sum(1)
        loss = loss + torch.where(rest > 0.0, rest * (torch.log(rest) - torch.log(mass)), 0.0)
        grad = grad - q * off * (rest / mass)[:, None]
    grad.scatter_add_(1, at, -p)
    grad = grad * (d["weight"] / T)[:, None]
    return dict(loss=torch.where(on, loss, 0.0), grad=grad.to(d["logits"].dtype))


def _plain_policy(case, d):
    T = case["T"]
    y, q, lse = _softmax(d["logits"], T)
    live = d["token"] >= 0
    t = d["token"].long().clamp(min=0)[:, None]
    lp = y.gather(1, t)[:, 0] - lse
    ratio, adv = torch.exp(lp - d["old"]), d["advantage"]
    kept = torch.minimum(torch.maximum(ratio, torch.full_like(ratio, 1.0 - CLIP_LOW)),
                         torch.full_like(ratio, 1.0 + CLIP_HIGH))
    loss = -torch.minimum(ratio * adv, kept * adv)
    clipped = ((adv > 0.0) & (ratio > 1.0 + CLIP_HIGH)) | ((adv < 0.0) & (ratio < 1.0 - CLIP_LOW))
    slope = torch.where(clipped, 0.0, -ratio * adv)
    kl = torch.zeros_like(lp)
    if case["ref"]:
        away = d["ref"] - lp
        kl = torch.exp(away) - away - 1.0
        loss = loss + KL * kl
        slope = slope + KL * (1.0 - torch.exp(away))
    c = torch.where(live, slope * d["weight"] / T, 0.0)[:, None]
    grad = -q * c
    grad.scatter_add_(1, t, c)
    return dict(loss=torch.where(live, loss, 0.0), logprob=torch.where(live, lp, 0.0), kl=torch.where(live, kl, 0.0),
                grad=grad.to(d["logits"].dtype))


def _sequence_of(start, rows):
    """The sequence that each row belongs to, 2 x pairs for rows behind the last."""
    return torch.searchsorted(start[1:].contiguous().long(), torch.arange(rows, device="cuda"), right=True)


def _plain_preference(case, d):
    T, pairs = case["T"], case["pairs"]
    y, q, lse = _softmax(d["logits"], T)
    rows = y.shape[0]
    live = d["token"] >= 0
    t = d["token"].long().clamp(min=0)[:, None]
    lp = torch.where(live, y.gather(1, t)[:, 0] - lse, 0.0)
    seq = _sequence_of(d["start"], rows)
    # sums of hundreds of terms, of which the loss takes small differences: in 64 bits
    total = torch.zeros(2 * pairs + 1, dtype=torch.float64, device="cuda").index_add_(0, seq, lp.double())[:-1]
    away = (total - d["ref"].double()).view(pairs, 2)
    h = BETA * (away[:, 0] - away[:, 1])
    eps = case["smooth"]
    up, down = 1.0 / (1.0 + torch.exp(-h)), 1.0 / (1.0 + torch.exp(h))
    loss = -(1.0 - eps) * torch.log(up) - eps * torch.log(down)
    slope = (eps * up - (1.0 - eps) * down) * BETA * d["weight"]
    each = torch.cat([torch.stack([slope, -slope], 1).view(-1), slope.new_zeros(1)])[seq].float()
    c = torch.where(live, each / T, 0.0)[:, None]
    grad = -q * c
    grad.scatter_add_(1, t, c)
    return dict(loss=loss.float(), logprob=total.float(), grad=grad.to(d["logits"].dtype))


_PLAIN = dict(logprobs=_plain_logprobs, top=_plain_top, distill=_plain_distill, policy=_plain_policy,
              preference=_plain_preference)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "preference":  # on average; the rows behind the sequences are not touched
        rows = 2 * case["pairs"] * (max(1, case["longest"] // 3) + case["longest"]) / 2
    else:
        rows = case["rows"]
    elements = rows * case["vocab"]
    read = elements * (1.0 - case.get("masked", 0.0))  # a masked row's logits are not needed
    nbytes = size * read + 16 * rows
    if case["kind"] == "top":
        nbytes += 8 * rows * case["k"]
    elif case["kind"] == "distill":
        nbytes += 8 * rows * case["k"]
    if case["kind"] != "top" and case.get("grad", True):
        nbytes += size * elements
    return {"bytes": nbytes, "flops": 4 * read}


# ---- the same results in 64 bits ----


def _exact_rows(x, T):
    z = x.double() / T
    lse = torch.logsumexp(z, 1)
    return z, lse


def _exact_tile(case, d, lo, hi, extra):
    kind, T = case["kind"], case["T"]
    z, lse = _exact_rows(d["logits"][lo:hi], T)
    n = hi - lo
    index = torch.arange(n, device="cuda")
    if kind == "top":
        return dict(value=torch.topk(d["logits"][lo:hi].double(), case["k"], dim=1).values, lse=lse)
    prob = torch.exp(z - lse[:, None])
    if kind == "distill":
        ids, valid = d["teacher_id"][lo:hi].long(), d["teacher_id"][lo:hi] >= 0
        weight = d["weight"][lo:hi].double()
        scaled = d["teacher_logit"][lo:hi].double() / T
        norm = d["teacher_lse"][lo:hi].double() if case["tail"] else \
            torch.logsumexp(scaled.masked_fill(~valid, -math.inf), 1)
        target = torch.exp(scaled - norm[:, None]).masked_fill(~valid, 0.0)
        spot = ids.clamp(min=0)
        dense = torch.zeros_like(z).scatter_add_(1, spot, target)
        member = torch.zeros_like(z).scatter_add_(1, spot, valid.double()) > 0
        loss = (torch.xlogy(target, target) - target * (z.gather(1, spot) - lse[:, None])).sum(1)
        if case["tail"]:
            rest = (1.0 - target.sum(1)).clamp(min=0.0)
            mass = prob.masked_fill(member, 0.0).sum(1)
            loss += torch.xlogy(rest, rest) - torch.xlogy(rest, mass)
            dense += torch.where(member, 0.0, prob * (rest / mass)[:, None])
        grad = (prob - dense) * (weight / T)[:, None]
        return dict(loss=torch.where(weight != 0.0, loss, 0.0), grad=grad)
    token = d["token"][lo:hi].long()
    live = token >= 0
    one = torch.zeros_like(z)
    one[index[live], token[live]] = 1.0
    lp = torch.where(live, z[index, token.clamp(min=0)] - lse, 0.0)
    if kind == "logprobs":
        entropy = -(prob * (z - lse[:, None])).sum(1)
        out = dict(logprob=lp, lse=torch.where(live, lse, 0.0), entropy=torch.where(live, entropy, 0.0))
        if case["grad"]:
            a, b = (torch.where(live, d[k][lo:hi].double(), 0.0)[:, None] for k in ("grad_logprob", "grad_entropy"))
            out["grad"] = (a * (one - prob) - b * prob * (z - lse[:, None] + entropy[:, None])) / T
        return out
    if kind == "policy":
        ratio, adv = torch.exp(lp - d["old"][lo:hi].double()), d["advantage"][lo:hi].double()
        inside = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
        loss, kl = torch.maximum(-ratio * adv, -inside * adv), torch.zeros_like(lp)
        slope = torch.where(-ratio * adv >= -inside * adv, -ratio * adv, 0.0)
        if case["ref"]:
            gap = d["ref"][lo:hi].double() - lp
            kl = torch.expm1(gap) - gap
            loss, slope = loss + KL * kl, slope - KL * torch.expm1(gap)
        c = torch.where(live, slope * d["weight"][lo:hi].double() / T, 0.0)
        return dict(loss=torch.where(live, loss, 0.0), logprob=lp, kl=torch.where(live, kl, 0.0),
                    grad=c[:, None] * (one - prob))
    if extra is None:  # first time over the rows: the log-probabilities alone
        return dict(lp=lp)
    return dict(grad=extra[lo:hi, None] * live[:, None].double() * (one - prob))


def _exact_all(case, d, extra=None):
    rows, parts = d["logits"].shape[0], []
    for lo in range(0, rows, TILE):
        parts.append(_exact_tile(case, d, lo, min(rows, lo + TILE), extra))
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "top":
        return dict(_exact_all(case, d), id=None)
    if case["kind"] != "preference":
        return _exact_all(case, d)
    lp = _exact_all(case, d)["lp"]
    start = d["start"].tolist()
    total = torch.stack([lp[a:b].sum() for a, b in zip(start[:-1], start[1:])])
    margin = BETA * ((total - d["ref"].double())[0::2] - (total - d["ref"].double())[1::2])
    eps = case["smooth"]
    loss = (1.0 - eps) * torch.nn.functional.softplus(-margin) + eps * torch.nn.functional.softplus(margin)
    slope = torch.sigmoid(margin) - (1.0 - eps)
    slope = slope * BETA * d["weight"].double() / case["T"]
    each = torch.zeros(d["logits"].shape[0], dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(start[:-1], start[1:])):
        each[a:b] = slope[i // 2] * (1.0 if i % 2 == 0 else -1.0)
    return dict(loss=loss, logprob=total, grad=_exact_all(case, d, each)["grad"])
