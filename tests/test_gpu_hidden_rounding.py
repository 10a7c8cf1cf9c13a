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


def spread(parts, rows):
    """`rows` gradients of one token: parts[k] in the k-th of equal shares of them, zeros elsewhere."""
    grad = torch.zeros((rows, 5), device=DEV)
    for k, v in enumerate(parts):
        grad[k * rows // len(parts)] = v
    return grad


@pytest.mark.parametrize("rows", [1, 40, 1_000])
@pytest.mark.parametrize("accumulate", [False, True])
def test_the_factor_of_a_table_gradient_is_a_binary32_number(ops, rows, accumulate):
    """Factors that binary32 rounds, or loses; sums of many rows past binary32 that the factor brings back."""
    token = torch.zeros(rows, dtype=torch.int32, device=DEV)

    def put(grad, scale):
        table = torch.full((2, 5), 0.0 if accumulate else 5.0, device=DEV)
        ops.embed_grad(grad, token, table_grad=table, scale=scale, accumulate=accumulate)
        assert (table[1] == 0.0).all()
        return table[0].double()

    def nearest(v):
        return torch.tensor(v, dtype=torch.float64).float().double().item()

    large, larger = nearest(1e20), nearest(2e38)
    for value, scale in ((large, 1e-46), (large, -1e-300), (3.0, 31.6), (-5.0, 31.6), (7.0, 1e-30), (1.0, 3.4e38),
                         (larger, 1.5), (larger, -1.0), (larger, 0.75), (nearest(1e-38), 1e30), (nearest(1e-44), 1.0),
                         (2.0, 0.0), (nearest(1.1), -1.0)):
        want = nearest(value * nearest(scale))
        assert (put(spread([value], rows), scale) == want).all(), (value, scale)
    for value in (math.inf, -math.inf, math.nan):
        for scale in (1.0, 31.6, -31.6, 1e-46, 0.0):
            got = put(spread([value], rows), scale)
            want = value * nearest(scale)  # inf * 0 is no number
            assert (got.isnan().all() if math.isnan(want) else (got == want).all()), (value, scale)
    if rows > 16:
        grad = torch.zeros((rows, 5), device=DEV)
        grad[[0, 17, 34]] = larger  # each of another part
        assert (put(grad, 0.25) == nearest(3 * larger * 0.25)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("table_dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_single_gradients_go_by_binary32_to_the_tables_type(ops, dtype, table_dtype, accumulate):
    """A token each, factors that binary32 holds: product, addition, type."""
    for k, scale in enumerate([1.0, 31.625, 1.0 + 2.0 ** -8 + 2.0 ** -20, -0.125, 2.0 ** -100, 2.0 ** 100]):
        g = gen(k)
        grad = (torch.randn((90, 131), generator=g, device=DEV) * 4.0).to(TYPES[dtype])
        token = torch.randperm(90, generator=g, device=DEV)
        old = torch.randn((90, 131), generator=g, device=DEV).to(TYPES[table_dtype])
        table = old.clone()
        ops.embed_grad(grad, token.int(), table_grad=table, scale=scale, accumulate=accumulate)
        want = torch.zeros((90, 131), device=DEV)
        want[token] = (grad.double() * scale).float()
        if accumulate:
            want += old.float()
        want = want.to(TYPES[table_dtype])
        assert torch.equal(table, want), (scale, (table != want).nonzero()[:3].tolist())
