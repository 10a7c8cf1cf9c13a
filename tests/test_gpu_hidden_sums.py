"""The weight's gradient of very many rows, to the bit: every row counts once."""
import pytest
import torch

from promptboot_amd.hidden import HIDDEN_MAX_ROWS, HiddenRows
from tests.test_gpu_hidden import DEV, TYPES, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    o = HiddenRows(0)
    yield o
    o.close()


# the most rows of each plan's smallest sizes; then sizes whose workgroups are as many as 768 rows each take, and one row less
SIZES = [(HIDDEN_MAX_ROWS, 9), (HIDDEN_MAX_ROWS, 512), (786_433, 100), (786_432, 100), (786_433, 1_025), (786_431, 1_025),
         (393_217, 2_049), (200_003, 513), (100_001, 4_097), (30_001, 8_193), (20_003, 16_385)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_the_weights_gradient_of_many_rows_is_exact(ops, rows, cols, dtype):
    """Rows of 1 and -1 have a root of 1, and products with whole numbers up to 7 are whole: sums of 1,048,576 of them are
    below 2^24, so binary32 holds each, in any order.  A row left out, or counted twice, shows."""
    g = gen(rows)
    t = TYPES[dtype]
    h = torch.empty((rows, cols), dtype=t, device=DEV)
    grad = torch.empty((rows, cols), dtype=t, device=DEV)
    want = torch.zeros(cols, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 26) // cols)
    for lo in range(0, rows, step):
        n = min(step, rows - lo)
        a = torch.randint(0, 2, (n, cols), generator=g, device=DEV, dtype=torch.int8) * 2 - 1
        b = torch.randint(-7, 8, (n, cols), generator=g, device=DEV, dtype=torch.int8)
        b[b == 0] = 1  # no row is without effect
        h[lo:lo + n], grad[lo:lo + n] = a.to(t), b.to(t)
        want += (a * b).float().sum(0).double()  # whole numbers below 2^24
    dw = torch.full((cols,), 5.0, device=DEV)
    ops.norm_grad(h, None, grad, eps=1e-75, grad_weight=dw)
    assert torch.equal(dw.double(), want), (dw.double() - want).abs().max().item()
    ops.norm_grad(h, None, grad, eps=1e-75, grad_weight=dw, accumulate=True)
    assert torch.equal(dw.double(), 2 * want)
    del h, grad
    torch.cuda.empty_cache()
