"""Decode steps whose log-probabilities fail."""
import pytest
import torch

from promptboot_amd import sampler as s
from tests.test_gpu_scores import make_logits, out

pytestmark = pytest.mark.gpu


def test_a_step_whose_scoring_is_refused_is_settled():
    """The step was enqueued: states, contexts and row states are those of a step without log-probabilities."""
    rows, limits = 4, [1, 3, 5, 5]
    made = [s.DecodeBatch([[1, 2, 3]] * rows, list(range(7, 7 + rows)), limits, device=0) for _ in range(2)]
    batch, plain = made

    class Refusing:
        def bind_token_logprobs(self, *a, **kw):
            def call():
                raise s.InferenceError(s._Error(status=s.DEVICE))
            return call

    for step in range(4):
        x, _ = make_logits(rows, s.VOCAB, "f32", seed=step)
        batch._scores = Refusing() if step in (0, 2) else None
        if step in (0, 2):
            with pytest.raises(s.InferenceError):
                batch.step(x, logprobs=out(rows))
        else:
            lp = out(rows)
            tokens = batch.step(x, logprobs=lp)
            assert ((torch.from_numpy(tokens.view("int32")) >= 0) == (lp.cpu() != 0)).all()
        plain.step(x)
        assert [a == b for a, b in zip(batch.sampling_states(), plain.sampling_states())] == [True] * rows
        assert all((a == b).all() for a, b in zip(batch.contexts(), plain.contexts()))
        assert (batch.row_state_host == plain.row_state_host).all()
    for b in made:
        b.close()
