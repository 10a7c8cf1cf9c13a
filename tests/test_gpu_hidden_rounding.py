"""Roundings of the operators on hidden-state rows: a product goes to binary32 and from there to the output's type."""
import math

import pytest
import torch

from promptboot_amd.hidden import HiddenRows
from tests.test_gpu_hidden import DEV, TYPES, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    o = HiddenRows(0)
    yield o
    o.close()


def same(got, want):
    bits = torch.int32 if got.dtype == torch.float32 else torch.int16
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan) and torch.equal(got.view(bits)[~nan], want.view(bits)[~nan])


SCALES = [1.0, 31.6, 1.0 + 2.0 ** -8 + 2.0 ** -40, 1.0 + 2.0 ** -8 - 2.0 ** -40, 1.0 + 2.0 ** -11 + 2.0 ** -40, -3.0, 0.0,
          1e-38, 1e-30, 1e30, -1e300]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_dtype", ["f32", "f16", "bf16"])
def test_the_embedding_rounds_to_binary32_and_then_to_its_type(ops, dtype, out_dtype):
    for k, scale in enumerate(SCALES):
        g = gen(k)
        table = torch.randn((40, 999), generator=g, device=DEV)
        table[::3] = torch.randint(-300, 300, table[::3].shape, generator=g, device=DEV)  # few digits: many halves
        table[1::3] *= 2.0 ** torch.randint(-12, 12, table[1::3].shape, generator=g, device=DEV)
        table[0, :8] = torch.tensor([1.0, -1.0, 0.0, -0.0, math.inf, -math.inf, math.nan, 3e38])
        table = table.to(TYPES[dtype])
        out = torch.empty(table.shape, dtype=TYPES[out_dtype], device=DEV)
        ops.embed(table, torch.arange(40, device=DEV).int(), out=out, scale=scale)
        same(out, (table.double() * scale).float().to(TYPES[out_dtype]))


def test_a_product_next_to_a_half_passes_through_it(ops):
    """1 + 2^-8 + 2^-40 is 1 + 2^-8 in binary32: a half of bfloat16's, which goes to the even number."""
    table, out = torch.ones((1, 8), dtype=torch.bfloat16, device=DEV), torch.empty((1, 8), dtype=torch.bfloat16, device=DEV)
    token = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.embed(table, token, out=out, scale=1.0 + 2.0 ** -8 + 2.0 ** -40)
    assert (out == 1.0).all()
    wide = torch.empty((1, 8), device=DEV)
    ops.embed(table, token, out=wide, scale=1.0 + 2.0 ** -8 + 2.0 ** -40)
    assert (wide == 1.0 + 2.0 ** -8).all()
    ops.embed(table, token, out=out, scale=1.0 + 2.0 ** -8 + 2.0 ** -20)
    assert (out == 1.0078125).all()
