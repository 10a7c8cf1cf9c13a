"""What a bound call's check raises, and that it enqueues nothing (no GPU)."""
import pytest
import torch

from promptboot_amd import hidden
from promptboot_amd import sampler as s
from tests.test_hidden_api import _Context, _Fake, f


def test_a_check_refuses_what_the_call_would():
    ops = hidden.HiddenRows(sampler=_Context())  # no real context: a call that got past the check would end the process
    b = torch.int8
    q, w, scale, ws, out = f(3, 8, dtype=b), f(5, 8, dtype=b), f(3), f(5), f(3, 5)
    ops.bind_matmul(q, scale, w, ws, out=out).check()
    ops.bind_quantize(f(3, 8), q=q, scale=scale).check()
    ops.bind_norm(f(3, 8), f(8), residual=f(3, 8), sum=f(3, 8), q=q, scale=scale).check()
    x = f(3, 8)
    ops.bind_norm(x, f(8), sum=x, q=q, scale=scale).check()
    for bad, status in ((ops.bind_matmul(q, scale, w, ws, out=out, bias=ws.data_ptr() + 2), s.ALIGNMENT),
                        (ops.bind_matmul(q, scale, w, scale.data_ptr() + 1, out=out), s.ALIGNMENT),
                        (ops.bind_matmul(q, scale, w, ws, out=out, bias=out.data_ptr()), s.STATE),
                        (ops.bind_norm(x, f(8), out=x, sum=x), s.STATE),
                        (ops.bind_norm(x, f(8), eps=0.0, out=x), s.ARITHMETIC),
                        (ops.bind_embed(f(9, 8), f(3), out=f(3, 8), scale=float("nan")), s.ARITHMETIC)):
        with pytest.raises(s.InferenceError) as e:
            bad.check()
        assert e.value.status == status
    ops.bind_quantize(_Fake(torch.zeros((0, 8))), q=f(0, 8, dtype=b), scale=f(0)).check()  # no rows
    call = ops.bind_quantize(f(3, 8), q=q, scale=scale)
    ops.close()
    with pytest.raises(ValueError, match="closed"):
        call.check()
