"""What a bound call uses lives as long as the call does."""
import gc
import weakref

import numpy as np
import pytest
import torch

from promptboot_amd import hip
from promptboot_amd import sampler as s
from promptboot_amd.scores import RowScorer
from tests import scores_reference as ref
from tests.test_gpu_scores import DEV, all_calls, ids_of, make_logits, out

pytestmark = pytest.mark.gpu


def test_bound_scores_keep_their_stream():
    rows, vocab = 6, 500
    x, g = make_logits(rows, vocab, "f32", seed=3)
    token = ids_of(x, g)
    sc = RowScorer(0)
    hs = hip.Stream()
    calls, o = all_calls(sc, x, token.int(), g, stream=hs)
    lives = weakref.ref(hs)
    del hs
    gc.collect()
    assert lives() is not None and lives().handle  # before anything is enqueued on it
    torch.cuda.synchronize()
    for c in calls:
        c()
    lives().synchronize()
    want = ref.logprobs(x, token)["logprob"]
    assert (o["lp"].double() - want).abs().max() < 1e-4
    for kind in range(len(calls)):  # each of them by itself
        assert any(b is lives() for b in calls[kind].buffers)
    del calls, c
    gc.collect()
    assert lives() is None
    sc.close()


def test_bound_samples_keep_their_stream_and_buffers():
    rows = 4
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 2.5, (rows, s.VOCAB)).astype(np.float32)
    smp = s.BatchSampler(0)
    token = hip.DeviceArray(rows, np.uint32)
    hs = hip.Stream()
    words = hip.DeviceArray.from_numpy(logits.view(np.uint32))
    r24 = hip.DeviceArray.from_numpy(rng.integers(0, 1 << 24, rows).astype(np.uint32))
    smp.sample(words, r24, token=token)
    hip.synchronize()
    want = token.numpy().copy()
    call = smp.bind_sample(words, r24, token=token, stream=hs)
    lives = [weakref.ref(v) for v in (hs, words, r24, smp)]
    del hs, words, r24, smp
    gc.collect()
    assert all(v() is not None for v in lives) and lives[0]().handle
    token.upload(np.zeros(rows, np.uint32))
    call()
    lives[0]().synchronize()
    assert (token.numpy() == want).all()
