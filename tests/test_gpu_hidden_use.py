"""Operators on hidden-state rows as they are used: decode steps through an 8-bit head, a training step from the
tokens to the table's gradient, captured graphs, two streams, and what a bound call keeps alive."""
import gc
import math
import weakref

import numpy as np
import pytest
import torch

from promptboot_amd import hip
from promptboot_amd import sampler as s
from promptboot_amd.hidden import HiddenRows
from promptboot_amd.scores import RowScorer
from tests import hidden_reference as ref
from tests import scores_reference
from tests.test_gpu_hidden import DEV, EPS, gen, make, make_bytes, near

pytestmark = pytest.mark.gpu


def head_of(g, cols):
    """A head whose logits of normed rows have a few far ahead of the others, as trained ones do."""
    weight = make_bytes(g, s.VOCAB, cols)
    return weight, torch.rand(s.VOCAB, generator=g, device=DEV) * 2e-3 / math.sqrt(cols) + 1e-4


@pytest.mark.parametrize("norm", [True, False])
def test_decode_steps_through_an_8_bit_head(norm):
    """Each step is its parts: the norm in 8 bits, the product, the decode step on those logits, the next embedding."""
    g = gen(4)
    rows, cols = 5, 100
    weight, weight_scale = head_of(g, cols)
    table = make(g, s.VOCAB, cols, "bf16")
    norm_weight = torch.rand(cols, generator=g, device=DEV) + 0.5
    args = ([[1, 2, 3]] * rows, list(range(11, 11 + rows)), [2, 4, 4, 4, 4])
    batch, plain = s.DecodeBatch(*args), s.DecodeBatch(*args)
    ops = HiddenRows(sampler=plain.sampler)
    hidden = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    batch.embed(table, out=hidden)  # nothing drawn yet
    torch.cuda.synchronize()
    assert (hidden == 0).all()
    hidden = make(g, rows, cols, "bf16")
    stream = make(g, rows, cols, "bf16")
    q, scale = torch.empty((rows, cols), dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    logits = torch.empty((rows, s.VOCAB), device=DEV)
    for step in range(4):
        lp = torch.full((rows,), 5.0, device=DEV)
        total = torch.empty_like(hidden)
        kw = dict(norm_weight=norm_weight, residual=stream, sum=total) if norm else {}
        torch.cuda.synchronize()
        tokens = batch.int8_step(hidden, weight, weight_scale, logprobs=lp, **kw)
        if norm:
            h = ref.rows_of(hidden, stream)
            assert torch.equal(total, h)
            ops.norm(h, norm_weight, q=q, scale=scale)
        else:
            ops.quantize(hidden, q=q, scale=scale)
        ops.matmul(q, scale, weight, weight_scale, out=logits)
        torch.cuda.synchronize()
        want = plain.step(logits)
        assert (tokens == want).all()
        live = torch.from_numpy(tokens.view(np.int32)).to(DEV).long()
        want_lp = scores_reference.logprobs(logits, live)["logprob"]
        assert (lp.double() - want_lp).abs().max() < 1e-4
        batch.embed(table, out=hidden)
        torch.cuda.synchronize()
        assert torch.equal(hidden, ref.embed(table, live, 1.0).to(hidden.dtype))
        if norm:
            stream = total
    assert all((a == b).all() for a, b in zip(batch.contexts(), plain.contexts()))
    assert (hidden[0] == 0).all() and tokens[0] == s.NO_TOKEN  # ended at its limit
    # a row that is not finite fails alone, without a draw
    batch2 = s.DecodeBatch([[1]] * rows, list(range(rows)), [3] * rows)
    hidden = make(g, rows, cols, "bf16")
    hidden[2, 7] = math.nan
    torch.cuda.synchronize()
    tokens = batch2.int8_step(hidden, weight, weight_scale, norm_weight=norm_weight if norm else None)
    assert tokens[2] == s.NO_TOKEN and batch2.row_state_host[2] == s.ROW_ERROR and (np.delete(tokens, 2) < s.VOCAB).all()
    assert [st.draws() for st in batch2.sampling_states()] == [1, 1, 0, 1, 1]
    # refusals leave the states as they are
    before = batch2.sampling_states()
    for bad in (lambda: batch2.int8_step(hidden[:3], weight, weight_scale),
                lambda: batch2.int8_step(hidden, weight[:100], weight_scale),
                lambda: batch2.int8_step(hidden, weight, weight_scale, residual=hidden),
                lambda: batch2.embed(table, out=hidden[:3]),
                lambda: batch2.int8_step(hidden, weight, weight_scale, logprobs=lp, logprob_temperature=0.0)):
        with pytest.raises(ValueError):
            bad()
    assert batch2.sampling_states() == before
    for b in (batch, plain, batch2):
        b.close()


def test_a_head_in_8_bits_is_near_the_head_it_is_made_from():
    """Rounded weights and rows: each is off by half a step of its channel's and row's largest at most."""
    g = gen(8)
    ops = HiddenRows(0)
    rows, channels, cols = 9, 1000, 300
    w, x = make(g, channels, cols, "bf16", spread=0.05), make(g, rows, cols, "bf16")
    wq, ws = torch.empty((channels, cols), dtype=torch.int8, device=DEV), torch.empty(channels, device=DEV)
    xq, xs = torch.empty((rows, cols), dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    out = torch.empty((rows, channels), device=DEV)
    ops.quantize(w, q=wq, scale=ws)
    ops.quantize(x, q=xq, scale=xs)
    ops.matmul(xq, xs, wq, ws, out=out)
    a, b = x.double(), w.double()
    dx, dw = xs.double()[:, None] / 2, ws.double()[:, None] / 2
    bound = dx @ b.abs().sum(1)[None, :] + a.abs().sum(1)[:, None] @ dw.t() + cols * (dx @ dw.t())
    assert ((out.double() - a @ b.t().contiguous()).abs() <= bound * 1.0001).all()
    ops.close()


def test_a_training_step_from_tokens_to_the_table():
    """embed -> norm -> a head -> policy loss -> the head's and the norm's gradient -> the table's: against autograd in 64 bits."""
    g = gen(5)
    ops, sc = HiddenRows(0), RowScorer(0)
    rows, vocab, cols, factor = 60, 200, 48, 3.0
    table = make(g, vocab, cols, "f32")
    norm_weight = torch.rand(cols, generator=g, device=DEV) + 0.5
    head = torch.randn((vocab, cols), generator=g, device=DEV) * 0.2
    token = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    token[::7] = -1  # padding
    target = torch.where(token >= 0, torch.randint(0, vocab, (rows,), generator=g, device=DEV), -1)
    old, adv = torch.full((rows,), -5.0, device=DEV), torch.randn(rows, generator=g, device=DEV)
    h, y = torch.empty((rows, cols), device=DEV), torch.empty((rows, cols), device=DEV)
    ops.embed(table, token.int(), out=h, scale=factor)
    ops.norm(h, norm_weight, eps=EPS, out=y)
    logits = y @ head.t().contiguous()
    loss, dlogits = torch.empty(rows, device=DEV), torch.empty_like(logits)
    sc.policy_loss(logits, target.int(), old, adv, loss=loss, grad=dlogits, clip_high=1e9, clip_low=1.0)
    dy = dlogits @ head
    dh, dw, dt = torch.empty_like(h), torch.empty(cols, device=DEV), torch.empty_like(table)
    ops.norm_grad(h, norm_weight, dy, eps=EPS, grad_h=dh, grad_weight=dw)
    ops.embed_grad(dh, token.int(), table_grad=dt, scale=factor)
    t64, w64 = (v.double().cpu().requires_grad_() for v in (table, norm_weight))
    live = (token >= 0).cpu()
    e = t64[token.cpu().clamp(min=0)] * factor * live[:, None]
    n = e / torch.sqrt((e * e).mean(1, keepdim=True) + EPS) * w64
    lp = torch.log_softmax(n @ head.double().cpu().t(), 1).gather(1, target.cpu().clamp(min=0)[:, None])[:, 0]
    total = (-torch.exp(lp - old.double().cpu()) * adv.double().cpu() * live).sum()
    total.backward()
    # binary32 chains of a few products of 48 terms: their errors add up to some 100 half steps of the largest terms
    assert (dt.cpu().double() - t64.grad).abs().max() < 1e-5 * t64.grad.abs().max()
    assert (dw.cpu().double() - w64.grad).abs().max() < 1e-5 * w64.grad.abs().max()
    assert abs(loss.double().sum().item() - total.item()) < 1e-4 * loss.double().abs().sum().item()
    ops.close()
    sc.close()


def all_calls(ops, g, stream=None, rows=70, cols=96, vocab=300):
    """Every operator, each on the one before: (bound calls, inputs, outputs)."""
    bf = torch.bfloat16
    i = dict(table=make(g, vocab, cols, "bf16"), token=torch.randint(-1, vocab, (rows,), generator=g, device=DEV).int(),
             residual=make(g, rows, cols, "bf16"), weight=torch.rand(cols, generator=g, device=DEV) + 0.5,
             dy=make(g, rows, cols, "bf16"), w=make(g, 200, cols, "bf16"))

    def new(*shape, dtype=bf):
        return torch.zeros(shape, dtype=dtype, device=DEV)

    o = dict(x=new(rows, cols), h=new(rows, cols), y=new(rows, cols), q=new(rows, cols, dtype=torch.int8),
             scale=new(rows, dtype=torch.float32), wq=new(200, cols, dtype=torch.int8), ws=new(200, dtype=torch.float32),
             out=new(rows, 200, dtype=torch.float32), dh=new(rows, cols), dw=new(cols, dtype=torch.float32),
             dt=new(vocab, cols, dtype=torch.float32))
    kw = dict(stream=stream)
    calls = [ops.bind_embed(i["table"], i["token"], out=o["x"], scale=2.0, **kw),
             ops.bind_norm(o["x"], i["weight"], residual=i["residual"], sum=o["h"], out=o["y"], q=o["q"],
                           scale=o["scale"], **kw),
             ops.bind_quantize(i["w"], q=o["wq"], scale=o["ws"], **kw),
             ops.bind_matmul(o["q"], o["scale"], o["wq"], o["ws"], out=o["out"], **kw),
             ops.bind_norm_grad(o["h"], i["weight"], i["dy"], grad_h=o["dh"], grad_weight=o["dw"], **kw),
             ops.bind_embed_grad(o["dh"], i["token"], table_grad=o["dt"], scale=2.0, **kw)]
    return calls, i, o


def renew(i, g, vocab=300):
    for k, v in i.items():
        if k == "token":
            v.copy_(torch.randint(-1, vocab, v.shape, generator=g, device=DEV))
        else:
            v.copy_(torch.randn(v.shape, generator=g, device=DEV))


def test_a_captured_graph_replays_on_new_inputs():
    g = gen(6)
    ops = HiddenRows(0)
    hs = hip.Stream()
    calls, i, o = all_calls(ops, g, stream=hs)
    torch.cuda.synchronize()
    for c in calls:
        c()
    hs.synchronize()
    graph = hip.Graph(hs)
    graph.begin()
    for c in calls:
        c()
    graph.end()
    for turn in range(4):
        renew(i, g)
        torch.cuda.synchronize()
        graph.launch()
        hs.synchronize()
        got = {k: v.clone() for k, v in o.items()}
        for v in o.values():
            v.zero_()
        if turn == 1:  # a workspace that grows leaves the graph's as it is
            ops.reserve(5000, 2000)
        torch.cuda.synchronize()
        for c in calls:
            c()
        hs.synchronize()
        for k in o:
            assert torch.equal(got[k], o[k]), (turn, k)
    graph.close()
    ops.close()


def test_two_contexts_on_two_streams():
    made = []
    for k in range(2):
        ops, hs = HiddenRows(0), hip.Stream()
        calls, i, o = all_calls(ops, gen(k), stream=hs, rows=3000, cols=640)
        made.append((ops, hs, calls, o))
    torch.cuda.synchronize()
    want = []
    for ops, hs, calls, o in made:
        for c in calls:
            c()
        hs.synchronize()
        want.append({k: v.clone() for k, v in o.items()})
        for v in o.values():
            v.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for pair in zip(made[0][2], made[1][2]):
            for c in pair:
                c()
    for _, hs, _, _ in made:
        hs.synchronize()
    for (ops, _, _, o), w in zip(made, want):
        assert all(torch.equal(o[k], w[k]) for k in o)
        ops.close()


def test_bound_calls_keep_their_stream_and_buffers():
    ops = HiddenRows(0)
    hs = hip.Stream()
    calls, i, o = all_calls(ops, gen(2), stream=hs)
    lives = weakref.ref(hs)
    kept = [weakref.ref(v) for v in i.values()]
    del hs, i
    gc.collect()
    assert lives() is not None and lives().handle and all(v() is not None for v in kept)
    for c in calls:
        assert any(b is lives() for b in c.buffers) and any(b is ops for b in c.buffers)
    torch.cuda.synchronize()
    for c in calls:
        c()
    lives().synchronize()
    del calls, c
    gc.collect()
    assert lives() is None and all(v() is None for v in kept)
    ops.close()


def test_device_arrays_without_another_framework():
    """Rows of numpy words: binary32 as it is, 16-bit words with their type's name."""
    rng = np.random.default_rng(3)
    ops = HiddenRows(0)
    d = hip.DeviceArray.from_numpy
    x = rng.normal(0, 1, (7, 50)).astype(np.float32)
    x16 = (x.view(np.uint32) >> 16).astype(np.uint16)  # bfloat16, truncated
    q, scale = hip.DeviceArray((7, 50), np.int8), hip.DeviceArray(7, np.float32)
    out = hip.DeviceArray((7, 50), np.uint32)
    ops.norm(d(x), q=q, scale=scale, out=out)
    t = torch.from_numpy(x)
    assert (q.numpy() == ref.quantized(t, None)[0].numpy()).all()
    got = torch.from_numpy(out.numpy().view(np.float32).copy())
    want = ref.norm(t, None, 1e-6)
    near(got, want, ref.norm_tolerance(want, torch.float32), "out")
    with pytest.raises(ValueError):
        ops.quantize(d(x16), q=q, scale=scale)
    ops.quantize(d(x16), q=q, scale=scale, dtype="bf16")
    t = torch.from_numpy(x16.view(np.int16).copy()).view(torch.bfloat16)
    assert (q.numpy() == ref.quantized(t, None)[0].numpy()).all()
    ops.close()
