"""Workspaces of the hidden-state rows' gradients: what the calls need, and no more than twice that."""
import ctypes

import pytest
import torch

from promptboot_amd import sampler as s
from promptboot_amd.hidden import HIDDEN_MAX_COLS, HIDDEN_MAX_ROWS, HiddenRows
from tests.test_gpu_hidden import DEV

pytestmark = pytest.mark.gpu

MIB = 1 << 20


def need(name, rows, cols):
    """What a call of this size reserves in a fresh context."""
    fresh = HiddenRows(0)
    e = s._Error()
    assert getattr(s.lib(), f"pb_context_reserve_{name}")(fresh.sampler._ctx, rows, cols, ctypes.byref(e)) == s.OK
    bytes_held = fresh.workspace_bytes()
    fresh.close()
    return bytes_held


@pytest.fixture
def ops():
    o = HiddenRows(0)
    yield o
    o.close()


def norm_grad(ops, rows, cols, dtype=torch.bfloat16):
    h = torch.zeros((rows, cols), dtype=dtype, device=DEV)
    ops.norm_grad(h, None, h, grad_weight=torch.empty(cols, device=DEV))


def embed_grad(ops, rows, cols, dtype=torch.bfloat16):
    grad, token = torch.zeros((rows, cols), dtype=dtype, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
    ops.embed_grad(grad, token, table_grad=torch.empty((3, cols), device=DEV))


def test_a_norms_gradient_reserves_its_own_need(ops):
    assert need("norm_grad", 65_536, 8_192) == 512 * 8_192 * 4
    norm_grad(ops, 65_536, 8_192)
    assert ops.workspace_bytes() == 512 * 8_192 * 4
    torch.cuda.empty_cache()


@pytest.mark.parametrize("order", [1, -1])
def test_a_long_narrow_call_and_a_short_wide_one_do_not_multiply(ops, order):
    """1,048,576 x 64 needs 50 MB and 16 x 32,768 less: their largest rows and columns together would need 16 GB."""
    sizes = [(HIDDEN_MAX_ROWS, 64), (16, HIDDEN_MAX_COLS)][::order]
    most = max(need(name, r, c) for r, c in sizes for name in ("embed_grad", "norm_grad"))
    assert most < 64 * MIB
    for rows, cols in sizes:
        embed_grad(ops, rows, cols)
        norm_grad(ops, rows, cols)
    assert most <= ops.workspace_bytes() <= 2 * most
    torch.cuda.empty_cache()


def test_growing_calls_grow_by_doubling(ops):
    held = [ops.workspace_bytes()]
    for rows in range(100, 4_000, 50):
        embed_grad(ops, rows, 600)
        norm_grad(ops, rows, 601)
        held.append(ops.workspace_bytes())
    sizes = sorted(set(held))
    assert sizes[0] == 0 and len(sizes) < 12
    assert all(b >= 2 * a for a, b in zip(sizes, sizes[1:]))
    assert sizes[-1] <= 2 * max(need("embed_grad", 4_000, 601), need("norm_grad", 4_000, 601))


def test_a_second_user_of_the_context_finds_what_is_there(ops):
    embed_grad(ops, 4_000, 600)
    have = ops.workspace_bytes()
    other = HiddenRows(sampler=ops.sampler)
    embed_grad(other, 3_999, 600)
    norm_grad(other, 100, 900)
    assert ops.workspace_bytes() == have
    other.close()
    embed_grad(ops, 100, 100)


def test_a_reservation_of_both_covers_both(ops):
    ops.reserve(5_000, 1_500)
    have = ops.workspace_bytes()
    for rows, cols in [(5_000, 1_500), (5_000, 512), (1, 1_500), (4_999, 1_025)]:
        embed_grad(ops, rows, cols)
        norm_grad(ops, rows, cols)
    assert ops.workspace_bytes() == have


def test_a_reservation_grows_to_what_the_largest_call_needs_at_most(ops):
    """A workspace of 10 GB that grows by a little: twice as much is more than any call needs."""
    rows, cols = HIDDEN_MAX_ROWS, 20_000
    ops._reserve("pb_context_reserve_embed_grad", rows, cols)
    held = ops.workspace_bytes()
    assert held == need("embed_grad", rows, cols) > 10_000 * MIB
    ops._reserve("pb_context_reserve_embed_grad", rows, cols + 1)
    assert held < ops.workspace_bytes() <= need("hidden", rows, HIDDEN_MAX_COLS)


def test_without_a_context_there_is_no_workspace():
    assert s.lib().pb_context_hidden_bytes(None) == 0
    closed = HiddenRows(0)
    closed.close()
    with pytest.raises(ValueError, match="closed"):
        closed.workspace_bytes()


@pytest.mark.parametrize("rows,cols", [(HIDDEN_MAX_ROWS, 9), (HIDDEN_MAX_ROWS, 512), (786_433, 100), (786_432, 100),
                                       (HIDDEN_MAX_ROWS, 513), (786_433, 1_025), (393_217, 2_049), (HIDDEN_MAX_ROWS, 32_768),
                                       (100_000, 20), (3, 9)])
def test_a_workgroup_adds_up_768_rows_at_most(rows, cols):
    """Each workgroup's sums of the weight's gradient are in 32 bits, so they hold 768 terms at most."""
    groups, left = divmod(need("norm_grad", rows, cols), cols * 4)
    at_once = 4 if cols <= 512 else 1  # rows that a workgroup takes at a time
    turns = -(-rows // at_once)
    assert left == 0 and -(-turns // groups) * at_once <= 768
