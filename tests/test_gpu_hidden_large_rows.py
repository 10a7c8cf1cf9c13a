"""Norms of rows next to the largest numbers, whose reciprocal roots are below binary32's normal range."""
import pytest
import torch

from promptboot_amd.hidden import HiddenRows
from tests import hidden_reference as ref
from tests.test_gpu_hidden import DEV, EPS, TYPES, gen, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    o = HiddenRows(0)
    yield o
    o.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(64, 100), (20, 777), (16, 3000), (8, 9000), (4, 20_000)])
def test_norms_of_rows_next_to_the_largest_numbers(ops, dtype, rows, cols):
    """1 / sqrt(mean) is below binary32's normal range there, where half of the smallest step is what it may be off by."""
    g = gen(rows)
    x = (1.0 + 2.0 * torch.rand((rows, cols), generator=g, device=DEV)) * 1e38
    x = (x * torch.where(torch.rand((rows, cols), generator=g, device=DEV) < 0.5, -1.0, 1.0)).to(TYPES[dtype])
    w = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[dtype])
    rstd = 1.0 / torch.sqrt((x.double() ** 2).mean(1, keepdim=True))
    assert (rstd < torch.finfo(torch.float32).smallest_normal).all()
    off = ref.tiny(torch.float32) / 2 / rstd  # of each product with it
    assert (off < 2.0 ** -21.9).all()
    for out_dtype in ("f32", "bf16"):
        out = torch.empty((rows, cols), dtype=TYPES[out_dtype], device=DEV)
        ops.norm(x, w, eps=EPS, out=out)
        want = ref.norm(x, w, EPS)
        near(out, want, ref.norm_tolerance(want, TYPES[out_dtype], w) + off * 1.01 * want.abs(), out_dtype)
    grad = (torch.randn((rows, cols), generator=g, device=DEV) * 2.0 ** 40).to(TYPES[dtype])  # (the result is normal)
    dh, dw = torch.empty_like(x), torch.empty(cols, device=DEV)
    ops.norm_grad(x, w, grad, eps=EPS, grad_h=dh, grad_weight=dw)
    want, want_weight = ref.norm_grad(x, w, grad, EPS)
    tol, tol_weight = ref.norm_grad_tolerances(x, w, grad, EPS, want, want_weight, TYPES[dtype])
    # of grad_h the factor times |g w| + |h k|, with |k| = |sum g w h| / cols rstd^2
    gw = grad.double() * w.double()
    terms = rstd * (gw.abs() + x.double().abs() * rstd * rstd * (gw * x.double()).abs().mean(1, keepdim=True))
    near(dh, want, tol + 1.01 * off * terms, "grad_h")
    near(dw, want_weight, tol_weight + 1.01 * (off * (grad.double() * x.double() * rstd).abs()).sum(0), "grad_weight")
