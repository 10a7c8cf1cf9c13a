"""Timed cases of the operators around a head: embedding rows, norms, 8-bit rows and their products.

A case is one call (or a forward and its gradient) of promptboot_amd.hidden.HiddenRows:

    embed   embed: the scaled table rows of a batch's tokens; with "grad" also embed_grad, the table's gradient.
    norm    norm: the residual's addition and the root-mean-square norm; "q8" leaves 8-bit rows with a scale each,
            "train" leaves the norm in the rows' type and takes its gradient (norm_grad).
    int8    matmul: 8-bit rows times 8-bit channels, with a scale for each of both, as logits or another layer's rows.

Everything is made on the GPU from the seed.  8-bit outputs come as the whole numbers they are, beside their scales:
which of two whole numbers a value goes to is worked out in 64 bits, so there is one answer.
"""
import math

import numpy as np
import torch

own = False

V = 151_936  # the model's vocabulary
NO_TOKEN = -1  # 0xffffffff as the int32 that torch holds
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
MOST_OPS = 4096 * V * 896  # of the largest product
MOST_ELEMENTS = 16_384 * 4_096  # of the largest norm


def listed():
    return [
        # a decode step of 40 conversations: the drawn tokens' rows, the next step's input
        dict(name="embed_40", kind="embed", rows=40, vocab=V, cols=896, dtype="bf16", scale=1.0, grad=False,
             grad_dtype="bf16", masked=0.0, pad=0),
        # a small training batch, 32 bits, another vocabulary, rows that start at any element; scaled by a width's root
        dict(name="embed_grad_700_odd", kind="embed", rows=700, vocab=50_257, cols=1_001, dtype="f32", scale=31.6,
             grad=True, grad_dtype="f32", masked=0.1, pad=3),
        # a training microbatch: most tokens frequent ones, padding without a token, the gradient summed in 32 bits
        dict(name="embed_grad_16384", kind="embed", rows=16_384, vocab=V, cols=896, dtype="bf16", scale=1.0, grad=True,
             grad_dtype="f32", masked=0.2, pad=0),
        # one conversation's decode step, before the head: latency
        dict(name="norm_q8_1", kind="norm", rows=1, cols=896, dtype="bf16", weight_dtype="bf16", q8=True, residual=True,
             pad=0),
        # a batch of decode steps of an odd width, in padded rows
        dict(name="norm_q8_70_odd", kind="norm", rows=70, cols=5_001, dtype="f16", weight_dtype="f32", q8=True,
             residual=True, pad=7),
        # a long prompt's rows before an 8-bit product
        dict(name="norm_q8_16384", kind="norm", rows=16_384, cols=4_096, dtype="bf16", weight_dtype="bf16", q8=True,
             residual=True, pad=0),
        # training on few rows of 32 bits, odd width
        dict(name="norm_train_300", kind="norm", rows=300, cols=1_001, dtype="f32", weight_dtype="f32", q8=False,
             residual=False, pad=0),
        # a training microbatch: forward and gradient
        dict(name="norm_train_8192", kind="norm", rows=8_192, cols=2_048, dtype="bf16", weight_dtype="bf16", q8=False,
             residual=True, pad=0),
        # one conversation's logits from an 8-bit head
        dict(name="int8_1", kind="int8", rows=1, n=V, cols=896, dtype="f32", bias=False, pad=0),
        # a decode step of 48 conversations through a wide layer
        dict(name="int8_48", kind="int8", rows=48, n=8_192, cols=8_192, dtype="bf16", bias=True, pad=0),
        # a ragged batch of rows, another vocabulary, an odd width
        dict(name="int8_333_odd", kind="int8", rows=333, n=50_257, cols=1_001, dtype="f16", bias=True, pad=5),
        # the largest: logits of a training batch's rows, for the losses
        dict(name="int8_4096", kind="int8", rows=4_096, n=V, cols=896, dtype="bf16", bias=False, pad=0),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "int8"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    pad = rng.choice([0, 0, 1, 8])
    if kind == "embed":
        cols = rng.choice([896, _log_uniform(rng, 64, 4_096)])
        vocab = rng.choice([V, _log_uniform(rng, 1_000, 200_000)])
        vocab = min(vocab, V * 896 // cols)  # a drawn table is no larger than the model's
        rows = min(_log_uniform(rng, 1, 16_384), 16_384 * 896 // cols)
        return dict(kind=kind, rows=rows, vocab=vocab, cols=cols, dtype=dtype, scale=rng.choice([1.0, 31.6]),
                    grad=rng.random() < 0.7, grad_dtype=rng.choice([dtype, "f32"]), masked=rng.choice([0.0, 0.1, 0.3]),
                    pad=pad)
    if kind == "norm":
        cols = rng.choice([896, _log_uniform(rng, 64, 16_384)])
        train = rng.random() < 0.5
        most = MOST_ELEMENTS * 2 // SIZES[dtype] // (4 if train else 1)
        return dict(kind=kind, rows=_log_uniform(rng, 1, min(16_384, most // cols)), cols=cols, dtype=dtype,
                    weight_dtype=rng.choice([dtype, "f32"]), q8=not train, residual=rng.random() < 0.7, pad=pad)
    cols = rng.choice([896, _log_uniform(rng, 64, 16_384)])
    n = min(rng.choice([V, _log_uniform(rng, 256, 200_000)]), V * 896 // cols)
    rows = min(_log_uniform(rng, 1, 4_096), MOST_OPS // (n * cols), 4_096 * V * 2 // (SIZES[dtype] * n))
    return dict(kind=kind, rows=max(1, rows), n=n, cols=cols, dtype=dtype, bias=rng.random() < 0.5, pad=pad)


# ---- inputs, on the GPU, from the seed alone ----


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rows(g, rows, cols, pad, dtype, spread=1.0):
    """N(0, spread^2) in rows of cols + pad elements."""
    full = torch.zeros((rows, cols + pad), dtype=TYPES[dtype], device="cuda")
    full[:, :cols] = _randn(g, rows, cols) * spread
    return full[:, :cols]


def _bytes(g, rows, cols, pad):
    """Rows of 8-bit whole numbers, as rounding to 8 bits leaves N(0, 1): 127 is near four deviations."""
    full = torch.zeros((rows, cols + pad), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // cols)
    for lo in range(0, rows, step):
        n = min(step, rows - lo)
        full[lo:lo + n, :cols] = (_randn(g, n, cols) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
    return full[:, :cols]


def _tokens(case, g):
    """Zipf tokens of exponent 1.1 by the inverse of its distribution, as promptboot_amd.workloads' histories have."""
    weight = torch.arange(1, case["vocab"] + 1, dtype=torch.float64, device="cuda").pow(-1.1)
    cdf = torch.cumsum(weight, 0)
    at = torch.rand(case["rows"], generator=g, device="cuda", dtype=torch.float64) * cdf[-1]
    token = torch.searchsorted(cdf, at).clamp(max=case["vocab"] - 1).int()
    return torch.where(_rand(g, case["rows"]) < case["masked"], NO_TOKEN, token)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, cols, pad = case["kind"], case["rows"], case["cols"], case["pad"]
    if kind == "embed":
        d = dict(table=_rows(g, case["vocab"], cols, pad, case["dtype"], 0.02), token=_tokens(case, g))
        if case["grad"]:
            d["grad"] = _rows(g, rows, cols, pad, case["dtype"])
        return d
    if kind == "norm":
        # a residual stream has a few columns that are much larger than the others
        d = dict(x=_rows(g, rows, cols, pad, case["dtype"]))
        d["weight"] = (1.0 + 0.2 * _randn(g, cols)).to(TYPES[case["weight_dtype"]])
        if case["residual"]:
            d["residual"] = _rows(g, rows, cols, pad, case["dtype"], 2.0)
            d["residual"][:, torch.randint(0, cols, (3,), generator=g, device="cuda")] *= 16.0
        if not case["q8"]:
            d["grad"] = _rows(g, rows, cols, pad, case["dtype"])
            if case["residual"]:
                d["grad_sum"] = _rows(g, rows, cols, pad, case["dtype"])
        return d
    d = dict(q=_bytes(g, rows, cols, pad), scale=_rand(g, rows) * 0.05 + 0.005)
    d["weight"] = _bytes(g, case["n"], cols, pad)
    d["weight_scale"] = _rand(g, case["n"]) * 1e-3 + 1e-4
    if case["bias"]:
        d["bias"] = _randn(g, case["n"])
    return d


def _zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    d = _inputs(case, seed)
    st = dict(case=case, d=d)
    if not own:
        return st
    from promptboot_amd.hidden import HiddenRows

    ops = HiddenRows(0)
    rows, cols, kind = case["rows"], case["cols"], case["kind"]
    dtype = TYPES[case["dtype"]]
    if kind == "embed":
        ops.reserve(rows, cols)
        out = dict(out=_zeros(rows, cols, dtype=dtype))
        calls = [ops.bind_embed(d["table"], d["token"], out=out["out"], scale=case["scale"])]
        if case["grad"]:
            out["grad"] = _zeros(case["vocab"], cols, dtype=TYPES[case["grad_dtype"]])
            calls.append(ops.bind_embed_grad(d["grad"], d["token"], table_grad=out["grad"], scale=case["scale"]))
    elif kind == "norm":
        ops.reserve(rows, cols)
        out = {}
        if case["residual"]:
            out["sum"] = _zeros(rows, cols, dtype=dtype)
        if case["q8"]:
            out.update(q=_zeros(rows, cols, dtype=torch.int8), scale=_zeros(rows))
            calls = [ops.bind_norm(d["x"], d["weight"], eps=EPS, residual=d.get("residual"), sum=out.get("sum"),
                                   q=out["q"], scale=out["scale"])]
        else:
            out.update(out=_zeros(rows, cols, dtype=dtype), grad_h=_zeros(rows, cols, dtype=dtype),
                       grad_weight=_zeros(cols))
            calls = [ops.bind_norm(d["x"], d["weight"], eps=EPS, residual=d.get("residual"), sum=out.get("sum"),
                                   out=out["out"]),
                     ops.bind_norm_grad(out["sum"] if case["residual"] else d["x"], d["weight"], d["grad"], eps=EPS,
                                        grad_sum=d.get("grad_sum"), grad_h=out["grad_h"],
                                        grad_weight=out["grad_weight"])]
    else:
        out = dict(out=_zeros(rows, case["n"], dtype=dtype))
        calls = [ops.bind_matmul(d["q"], d["scale"], d["weight"], d["weight_scale"], out=out["out"],
                                 bias=d.get("bias"))]
    return dict(st, ops=ops, calls=calls, out=out)


def run(state):
    if not own:
        return _PLAIN[state["case"]["kind"]](state["case"], state["d"])
    for call in state["calls"]:
        call()
    return state["out"]


# ---- the plain form ----


def _plain_embed(case, d):
    live = d["token"] >= 0
    t = d["token"].long().clamp(min=0)
    rows = d["table"][t].float() * case["scale"]
    out = dict(out=torch.where(live[:, None], rows, 0.0).to(d["table"].dtype))
    if case["grad"]:
        total = torch.zeros((case["vocab"], case["cols"]), device="cuda")
        total.index_add_(0, t, torch.where(live[:, None], d["grad"].float(), 0.0))
        out["grad"] = (total * case["scale"]).to(TYPES[case["grad_dtype"]])
    return out


def _plain_norm(case, d):
    x, out = d["x"], {}
    h = x
    if case["residual"]:
        h = out["sum"] = (x.float() + d["residual"].float()).to(x.dtype)
    f, w = h.float(), d["weight"].float()
    rstd = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)
    if case["q8"]:
        p = h.double() * d["weight"].double()  # which whole number is nearer, at the border: in 64 bits
        top = p.abs().amax(1, keepdim=True)
        out["q"] = torch.where(top > 0.0, torch.round(p * 127.0 / top), 0.0).to(torch.int8)
        out["scale"] = (rstd * (top / 127.0).float())[:, 0]
        return out
    out["out"] = (f * rstd * w).to(x.dtype)
    g = d["grad"].float()
    wg = g * w
    grad = rstd * (wg - f * (rstd * rstd * (wg * f).mean(1, keepdim=True)))
    if case["residual"]:
        grad = grad + d["grad_sum"].float()
    out["grad_h"] = grad.to(x.dtype)
    out["grad_weight"] = (g * (f * rstd)).sum(0)
    return out


def _plain_int8(case, d):
    y = d["q"].float() @ d["weight"].float().t()
    y = y * d["scale"][:, None] * d["weight_scale"]
    if case["bias"]:
        y = y + d["bias"]
    return dict(out=y.to(TYPES[case["dtype"]]))


_PLAIN = dict(embed=_plain_embed, norm=_plain_norm, int8=_plain_int8)


def _distinct(case):
    """How many different tokens a batch of the case holds, on average."""
    weight = np.arange(1, case["vocab"] + 1, dtype=np.float64) ** -1.1
    share = (1.0 - case["masked"]) * weight / weight.sum()
    return float(-np.expm1(case["rows"] * np.log1p(-share)).sum())


def work(case):
    s, rows, cols = SIZES[case["dtype"]], case["rows"], case["cols"]
    if case["kind"] == "embed":
        live = rows * (1.0 - case["masked"])
        nbytes = 4 * rows + cols * s * (_distinct(case) + rows)
        if case["grad"]:
            nbytes += cols * (s * live + SIZES[case["grad_dtype"]] * case["vocab"])
        return {"bytes": nbytes, "flops": cols * live * (2 if case["grad"] else 1)}
    if case["kind"] == "norm":
        each = s + (2 * s if case["residual"] else 0)
        if case["q8"]:
            each += 1
        else:  # the norm; then the sum and its gradients in, the rows' gradient out
            each += s + 3 * s + (s if case["residual"] else 0)
        return {"bytes": rows * cols * each, "flops": rows * cols * (6 if case["q8"] else 16)}
    nbytes = (rows + case["n"]) * cols + 4 * (rows + case["n"]) + s * rows * case["n"]
    return {"bytes": nbytes, "flops": 2 * rows * case["n"] * cols}


# ---- the same results in 64 bits ----


def _exact_embed(case, d):
    idx = d["token"].long()
    live = torch.nonzero(idx >= 0)[:, 0]
    out = torch.zeros((case["rows"], case["cols"]), dtype=torch.float64, device="cuda")
    out[live] = d["table"].index_select(0, idx[live]).double().mul_(case["scale"])
    res = dict(out=out)
    if case["grad"]:
        # by token in order, the rows of each added up
        order = torch.argsort(idx[live], stable=True)
        ids, n = torch.unique_consecutive(idx[live][order], return_counts=True)
        segment = torch.repeat_interleave(torch.arange(ids.numel(), device="cuda"), n)
        table = torch.zeros((case["vocab"], case["cols"]), dtype=torch.float64, device="cuda")
        sums = torch.zeros((ids.numel(), case["cols"]), dtype=torch.float64, device="cuda")
        sums.index_add_(0, segment, d["grad"][live[order]].double())
        table[ids] = sums * case["scale"]
        res["grad"] = table
    return res


def _exact_norm(case, d):
    res, total = {}, d["x"].double()
    if case["residual"]:
        res["sum"] = total + d["residual"].double()
        total = res["sum"].to(d["x"].dtype).double()  # the rows are the sum as it is held
    w = d["weight"].double()
    inv = torch.rsqrt(total.pow(2).sum(1) / case["cols"] + EPS)[:, None]
    unit = total * inv
    if case["q8"]:
        res["q"] = None
        res["scale"] = torch.linalg.vector_norm(unit * w, ord=math.inf, dim=1) / 127.0
        return res
    res["out"] = unit * w
    dy = d["grad"].double()
    dn = dy * w
    along = torch.einsum("rc,rc->r", dn, unit)[:, None] / case["cols"]
    res["grad_h"] = inv * (dn - unit * along)
    if case["residual"]:
        res["grad_h"] = res["grad_h"] + d["grad_sum"].double()
    res["grad_weight"] = torch.einsum("rc,rc->c", dy, unit)
    return res


def _exact_int8(case, d):
    # sums of 1,024 products of 8-bit numbers are below 2^24, so whole in 32 bits; more of them are added in 64
    acc = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device="cuda")
    for lo in range(0, case["cols"], 1024):
        a, b = d["q"][:, lo:lo + 1024].float(), d["weight"][:, lo:lo + 1024].float()
        acc += torch.mm(a, b.t().contiguous())
    acc.mul_(torch.outer(d["scale"].double(), d["weight_scale"].double()))
    return dict(out=acc + d["bias"].double() if case["bias"] else acc)


def exact(case, seed):
    return dict(embed=_exact_embed, norm=_exact_norm, int8=_exact_int8)[case["kind"]](case, _inputs(case, seed))
