"""Refused steps through an 8-bit head: nothing that the caller holds changes, so the step can be taken again."""
import pytest
import torch

from promptboot_amd import sampler as s
from tests.test_gpu_hidden import DEV, gen, make, make_bytes

pytestmark = pytest.mark.gpu

ROWS, COLS = 3, 96


@pytest.fixture(scope="module")
def head():
    g = gen(21)
    return make_bytes(g, s.VOCAB, COLS), torch.rand(s.VOCAB, generator=g, device=DEV) * 1e-3


def new_batch(**kw):
    return s.DecodeBatch([[1, 2, 3]] * ROWS, [5, 6, 7], [4] * ROWS, **kw)


REFUSED = {
    "a short bias": dict(bias=("zeros", 7)),
    "a bias at no word": dict(bias=("address", (1 << 50) + 2)),
    "a short scale": dict(weight_scale=("zeros", s.VOCAB - 1)),
    "a scale at no word": dict(weight_scale=("address", (1 << 50) + 1)),
    "an unsigned head": dict(weight="unsigned"),
    "a short buffer of log-probabilities": dict(logprobs=("zeros", ROWS - 1)),
    "a temperature of 0": dict(logprobs=("zeros", ROWS), logprob_temperature=0.0),
}


@pytest.mark.parametrize("place", ["residual", "hidden", "apart", "no norm"])
@pytest.mark.parametrize("what", REFUSED)
def test_a_refused_step_leaves_everything_as_it_was(head, what, place):
    g = gen(1)
    weight, weight_scale = head
    hidden, residual = make(g, ROWS, COLS, "bf16"), make(g, ROWS, COLS, "bf16")
    gamma, apart = torch.ones(COLS, device=DEV), torch.full((ROWS, COLS), 5.0, dtype=torch.bfloat16, device=DEV)
    norm = {} if place == "no norm" else dict(
        norm_weight=gamma, residual=residual, sum={"residual": residual, "hidden": hidden, "apart": apart}[place])
    kw = {}
    for k, v in REFUSED[what].items():
        if isinstance(v, tuple):
            v = torch.zeros(v[1], device=DEV) if v[0] == "zeros" else v[1]
        elif v == "unsigned":
            v = weight.view(torch.uint8)
        kw[k] = v
    batch = new_batch()
    batch.int8_step(hidden.clone(), weight, weight_scale)  # the buffers of a step are there
    before = [t.clone() for t in (hidden, residual, apart)]
    states, contexts = batch.sampling_states(), [c.tolist() for c in batch.contexts()]
    args = dict(dict(weight=weight, weight_scale=weight_scale), **kw)
    with pytest.raises((ValueError, s.InferenceError)):
        batch.int8_step(hidden, **norm, **args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (hidden, residual, apart)))
    assert batch.sampling_states() == states and [c.tolist() for c in batch.contexts()] == contexts
    # taken again, it is the step that was meant
    batch.int8_step(hidden, weight, weight_scale, **norm)
    want = before[0] + before[1]
    if norm:
        assert torch.equal(norm["sum"], want)
    assert [st.draws() for st in batch.sampling_states()] == [2] * ROWS
    batch.close()


def test_a_forced_slice_plan_has_its_workspace(head):
    """A sampler of many slices a row takes a step of many rows without a reservation of the caller's."""
    weight, weight_scale = head
    rows, sampler = 500, s.BatchSampler(0, segments=64)
    args = ([[1, 2]] * rows, list(range(rows)), [4] * rows)
    batch, plain = s.DecodeBatch(*args, sampler=sampler), s.DecodeBatch(*args)
    hidden, residual = make(gen(2), rows, COLS, "bf16"), make(gen(3), rows, COLS, "bf16")
    want, gamma = hidden + residual, torch.ones(COLS, device=DEV)
    expect = plain.int8_step(hidden, weight, weight_scale, norm_weight=gamma, residual=residual.clone())
    tokens = batch.int8_step(hidden, weight, weight_scale, norm_weight=gamma, residual=residual, sum=residual)
    assert torch.equal(residual, want) and (tokens == expect).all()
    for b in (batch, plain, sampler):
        b.close()


@pytest.mark.parametrize("closed", ["batch", "sampler"])
def test_a_closed_batch_refuses(head, closed):
    weight, weight_scale = head
    sampler = s.BatchSampler(0) if closed == "sampler" else None
    batch = new_batch(sampler=sampler)
    hidden, table = make(gen(1), ROWS, COLS, "bf16"), make(gen(2), s.VOCAB, COLS, "bf16")
    residual, out = make(gen(3), ROWS, COLS, "bf16"), torch.full((ROWS, COLS), 5.0, dtype=torch.bfloat16, device=DEV)
    logits, logprobs = torch.zeros((ROWS, s.VOCAB), device=DEV), torch.full((ROWS,), 5.0, device=DEV)
    packed, rows_32 = torch.zeros(1, dtype=torch.uint8, device=DEV), torch.zeros((ROWS, COLS), device=DEV)
    before = residual.clone()
    states = batch.sampling_states()
    (batch if closed == "batch" else sampler).close()
    torch.cuda.synchronize()
    for bad in (lambda: batch.embed(table, out=out),
                lambda: batch.int8_step(hidden, weight, weight_scale),
                lambda: batch.int8_step(hidden, weight, weight_scale, norm_weight=torch.ones(COLS, device=DEV),
                                        residual=residual, sum=residual),
                lambda: batch.step(logits), lambda: batch.step(logits, logprobs=logprobs),
                lambda: batch.lmhead_step(packed, rows_32), lambda: batch.lmhead_step(packed, rows_32, q8=True)):
        with pytest.raises(ValueError, match="closed"):
            bad()
    torch.cuda.synchronize()
    assert torch.equal(residual, before) and (out == 5.0).all() and (logprobs == 5.0).all()
    assert batch.sampling_states() == states
