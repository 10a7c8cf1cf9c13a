"""Which workspaces calls on hidden-state rows reserve (no GPU)."""
import ctypes

import pytest

from promptboot_amd import hidden
from promptboot_amd import sampler as s
from tests.test_hidden_api import f, rows  # noqa: F401  (a fixture)


def test_each_gradient_reserves_its_own_size(rows):  # noqa: F811
    rows.bind_embed_grad(f(700, 8), f(700), table_grad=f(9, 8))
    rows.bind_norm_grad(f(3, 900), f(900), f(3, 900), grad_weight=f(900))
    rows.bind_norm_grad(f(3, 900), f(900), f(3, 900), grad_h=f(3, 900))  # needs none
    rows.bind_norm(f(3, 8), f(8), out=f(3, 8))
    assert [(name, a[1:3]) for name, a in rows.made] == [("pb_context_reserve_embed_grad", (700, 8)),
                                                         ("pb_context_reserve_norm_grad", (3, 900))]
    assert rows._reserved == (0, 0)
    rows.reserve(10, 20)
    rows.reserve(10, 20)
    assert [(name, a[1:3]) for name, a in rows.made[2:]] == [("pb_context_reserve_hidden", (10, 20))]


@pytest.mark.parametrize("name", ["hidden", "embed_grad", "norm_grad"])
def test_reservations_are_checked(name):
    fn = getattr(s.lib(), f"pb_context_reserve_{name}")
    for rows, cols, status in [(1, 0, s.CAPACITY), (1, hidden.HIDDEN_MAX_COLS + 1, s.CAPACITY),
                               (hidden.HIDDEN_MAX_ROWS + 1, 10, s.CAPACITY), (1, 10, s.STATE), (0, 10, s.STATE)]:
        e = s._Error()
        assert fn(None, rows, cols, ctypes.byref(e)) == status and e.status == status
    assert fn(None, 1, 0, None) == s.CAPACITY  # err may be NULL


def test_no_context_holds_nothing():
    assert s.lib().pb_context_hidden_bytes(None) == 0
