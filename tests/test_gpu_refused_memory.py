"""Memory that the device does not have is refused once: the next call, of this or another library, is none the wiser."""
import ctypes

import numpy as np
import pytest
import torch

from promptboot_amd import hip
from promptboot_amd import sampler as s
from promptboot_amd.hidden import HiddenRows
from promptboot_amd.scores import RowScorer

pytestmark = pytest.mark.gpu


def too_much(refuse):
    if refuse == "reservation":
        sampler = s.BatchSampler(0, segments=32)
        with pytest.raises(s.InferenceError):
            sampler.reserve(0xFFFFFFFF)  # 22 TB
        sampler.close()
    else:
        with pytest.raises(hip.HipError):
            hip.DeviceArray(1 << 45, np.uint8)  # 35 TB


@pytest.mark.parametrize("refuse", ["reservation", "array"])
@pytest.mark.parametrize("then", ["torch", "hidden rows", "scores", "sample", "bare"])
def test_what_was_refused_is_no_later_calls_error(refuse, then):
    ops = HiddenRows(0)
    scorer = RowScorer(sampler=ops.sampler)
    x, out = torch.ones((5, 100), device="cuda"), torch.empty((5, 100), device="cuda")
    logits, r24 = torch.zeros((2, s.VOCAB), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    token = torch.zeros(2, dtype=torch.int32, device="cuda")
    lp = torch.empty(2, device="cuda")
    scorer.token_logprobs(logits, token, logprob=lp)
    torch.cuda.synchronize()
    too_much(refuse)
    if then == "torch":
        out.fill_(1.0)
    elif then == "hidden rows":
        ops.norm(x, None, out=out)
    elif then == "scores":
        scorer.token_logprobs(logits, token, logprob=lp)
    elif then == "sample":
        ops.sampler.sample(logits, r24, token=token)
    else:
        fn = ctypes.CDLL("libamdhip64.so.7").hipGetLastError
        assert fn() == 0
    torch.cuda.synchronize()
    if then == "hidden rows":
        assert (out - 1.0).abs().max() < 1e-6
    ops.close()
