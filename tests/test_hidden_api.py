"""Refusals of the operators on hidden-state rows, and their formulas' gradients against differences (no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from promptboot_amd import hidden, scores
from promptboot_amd import sampler as s
from tests import hidden_reference as ref

A = 1 << 20  # addresses nobody reads: every refusal comes before the GPU
FAR = 1 << 24  # apart from each other


def at(k):
    return A + k * FAR


CALLS = {
    "embed": ("pb_embed_rows",
              dict(table=at(0), dtype=scores.F32, vocab=50, cols=100, table_ld=128, rows=4, token=at(1), factor=1.0,
                   out=at(2), out_dtype=scores.F32, out_ld=128, err=at(3))),
    "embed_grad": ("pb_embed_rows_grad",
                   dict(grad=at(0), dtype=scores.F32, vocab=50, cols=100, grad_ld=128, rows=4, token=at(1), factor=1.0,
                        accumulate=0, table=at(2), table_dtype=scores.F32, table_ld=128)),
    "norm": ("pb_norm_rows",
             dict(x=at(0), dtype=scores.F32, cols=100, x_ld=128, rows=4, residual=at(1), residual_ld=128, weight=at(2),
                  weight_dtype=scores.F32, eps=1e-6, sum=at(3), sum_ld=128, out=at(4), out_dtype=scores.F32, out_ld=128,
                  q=at(5), q_ld=128, scale=at(6), err=at(7))),
    "norm_grad": ("pb_norm_rows_grad",
                  dict(h=at(0), dtype=scores.F32, cols=100, h_ld=128, rows=4, weight=at(1), weight_dtype=scores.F32,
                       eps=1e-6, grad=at(2), grad_dtype=scores.F32, grad_ld=128, grad_sum=at(3), grad_sum_ld=128,
                       grad_h=at(4), grad_h_ld=128, grad_weight=at(5), accumulate=0)),
    "quantize": ("pb_quantize_rows",
                 dict(x=at(0), dtype=scores.F32, cols=100, x_ld=128, rows=4, q=at(1), q_ld=128, scale=at(2), err=at(3))),
    "matmul": ("pb_int8_matmul",
               dict(q=at(0), q_ld=128, scale=at(1), rows=4, cols=100, weight=at(2), weight_ld=128, weight_scale=at(3),
                    channels=50, bias=at(4), out=at(5), out_dtype=scores.F32, out_ld=128)),
}


def call(name, **kw):
    """A call without a context: (status, error record)."""
    fn, given = CALLS[name]
    assert set(kw) <= set(given), (name, kw)
    e = s._Error()
    return getattr(s.lib(), fn)(None, *{**given, **kw}.values(), None, ctypes.byref(e)), e


def no_context(st, e):
    return st == s.STATE and e.status == s.STATE and e.needed == 1


@pytest.mark.parametrize("name", CALLS)
def test_sizes_are_checked(name):
    given = CALLS[name][1]
    assert no_context(*call(name))  # nothing else is wrong: the missing context is
    cases = [(dict(cols=0), s.CAPACITY), (dict(cols=hidden.HIDDEN_MAX_COLS + 1), s.CAPACITY),
             (dict(rows=hidden.HIDDEN_MAX_ROWS + 1), s.CAPACITY)]
    for k in given:
        if k.endswith("_ld"):
            cols = 50 if (name, k) == ("matmul", "out_ld") else 100
            cases += [({k: cols - 1}, s.CAPACITY), ({k: 1 << 38}, s.CAPACITY)]
        if k.endswith("dtype"):
            cases += [({k: 3}, s.STATE)]
        if k in ("vocab", "channels"):
            cases += [({k: 0}, s.CAPACITY), ({k: scores.SCORE_MAX_VOCAB + 1}, s.CAPACITY)]
        if k == "eps":
            cases += [({k: v}, s.ARITHMETIC) for v in (0.0, -1e-6, math.nan, math.inf)]
        if k == "factor":
            cases += [({k: v}, s.ARITHMETIC) for v in (math.nan, math.inf, -math.inf)]
    for kw, status in cases:
        st, e = call(name, **kw)
        assert st == status and e.status == status and not no_context(st, e), (kw, st)
    if name == "embed_grad":
        assert call(name, factor=1e39)[0] == s.ARITHMETIC  # past binary32
    for k, v in given.items():  # widest types and largest sizes that are taken
        if k == "cols":
            lds = {n: 1 << 20 for n in given if n.endswith("_ld")}
            apart = {n: (1 << 50) + i * (1 << 44) for i, n in enumerate(m for m in given if given[m] in map(at, range(8)))}
            big = dict(cols=hidden.HIDDEN_MAX_COLS, rows=hidden.HIDDEN_MAX_ROWS, **lds, **apart)
            assert no_context(*call(name, **big)), name


REQUIRED = {"embed": ["table", "token", "out"], "embed_grad": ["grad", "token", "table"], "norm": ["x", "scale"],
            "norm_grad": ["h", "grad"], "quantize": ["x", "q", "scale"],
            "matmul": ["q", "scale", "weight", "weight_scale", "out"]}
OPTIONAL = {"embed": ["err"], "embed_grad": [], "norm": ["residual", "weight", "sum", "out", "err"],
            "norm_grad": ["weight", "grad_sum", "grad_h", "grad_weight"], "quantize": ["err"], "matmul": ["bias"]}


@pytest.mark.parametrize("name", CALLS)
def test_buffers_are_checked(name):
    for k in REQUIRED[name]:
        st, e = call(name, **{k: None})
        assert st == s.CAPACITY and e.detail == (4 << 32 | 3), k
    for k in OPTIONAL[name]:
        assert no_context(*call(name, **{k: None})), k
    given = CALLS[name][1]
    for k, v in given.items():
        if v in map(at, range(8)) and not (k == "q" or (name, k) == ("matmul", "weight")):  # bytes start anywhere
            assert call(name, **{k: v + 2})[0] == s.ALIGNMENT, k
    if "err" in given:
        assert call(name, err=given["err"] + 4)[0] == s.ALIGNMENT
    rows = dict(rows=0, **{k: None for k in REQUIRED[name]})
    if name == "norm_grad":
        assert no_context(*call(name, **rows))  # the weight's gradient is written all the same
        assert call(name, **rows, grad_weight=None)[0] == s.OK and call(name, **rows, accumulate=1)[0] == s.OK
    elif name == "embed_grad":
        assert call(name, **rows)[0] == s.CAPACITY and call(name, **rows, accumulate=1)[0] == s.OK
    else:
        assert call(name, **rows)[0] == s.OK
    if name == "norm":
        assert call(name, out=None, q=None, scale=None)[0] == s.CAPACITY
        assert no_context(*call(name, q=None, scale=None))
    if name == "norm_grad":
        assert call(name, grad_h=None, grad_weight=None)[0] == s.CAPACITY


# output -> the inputs in whose place it may lie
PLACES = {"embed": {"out": [], "err": []}, "embed_grad": {"table": []},
          "norm": {"sum": ["x", "residual"], "out": ["x", "residual"], "q": [], "scale": [], "err": []},
          "norm_grad": {"grad_h": ["h", "grad", "grad_sum"], "grad_weight": []},
          "quantize": {"q": [], "scale": [], "err": []}, "matmul": {"out": []}}


@pytest.mark.parametrize("name", CALLS)
def test_outputs_share_nothing(name):
    given = CALLS[name][1]
    buffers = [k for k, v in given.items() if v in map(at, range(8))]
    for o, places in PLACES[name].items():
        for other in buffers:
            if other == o:
                continue
            st, e = call(name, **{o: given[other]})
            if other in places:
                assert no_context(st, e), (o, other)
            else:
                assert st == s.STATE and e.detail == (4 << 32 | 9), (o, other)
            step = 8  # every buffer's alignment
            st, e = call(name, **{o: given[other] + step})
            assert st == s.STATE and e.detail == (4 << 32 | 9), (o, other)
        ld = {"sum": "sum_ld", "grad_h": "grad_h_ld", "out": "out_ld"}.get(o)
        for other in places:  # at another distance of rows, or of another type, it is no place
            assert call(name, **{o: given[other], ld: 256})[1].detail == (4 << 32 | 9)
            if o == "out":
                assert call(name, **{o: given[other], "out_dtype": scores.BF16})[1].detail == (4 << 32 | 9)
            if other == "grad":
                assert call(name, **{o: given[other], "grad_dtype": scores.BF16})[1].detail == (4 << 32 | 9)
    if name == "norm":  # two outputs in one place
        assert call(name, sum=given["x"], out=given["x"])[1].detail == (4 << 32 | 9)
        assert no_context(*call(name, sum=given["x"], out=given["residual"]))


def test_rows_may_lie_between_each_other():
    """Columns of one buffer, and every other row of it."""
    x = dict(x=at(0), x_ld=256, residual=None, sum=None, out_ld=256)
    for shift, ok in [(100 * 4, True), (99 * 4, False), (156 * 4, True), (157 * 4, False), (-156 * 4, True),
                      (-157 * 4, False), (-100 * 4, True), (-99 * 4, False), ((256 * 3 + 99) * 4, False),
                      ((256 * 3 + 100) * 4, True), (256 * 4 * 4, True), ((256 * 4 - 57) * 4, True), (256 * 4, False)]:
        st, e = call("norm", **x, out=at(0) + shift)
        assert no_context(st, e) == ok and (ok or st == s.STATE), shift
    # of two distances the ranges they span are compared
    assert call("norm", **{**x, "out_ld": 260}, out=at(0) + 400)[0] == s.STATE


def test_reservation_is_checked():
    fn = s.lib().pb_context_reserve_hidden
    for rows, cols, status in [(1, 0, s.CAPACITY), (1, hidden.HIDDEN_MAX_COLS + 1, s.CAPACITY),
                               (hidden.HIDDEN_MAX_ROWS + 1, 10, s.CAPACITY), (1, 10, s.STATE)]:
        e = s._Error()
        assert fn(None, rows, cols, ctypes.byref(e)) == status and e.status == status
    assert fn(None, 1, 0, None) == s.CAPACITY  # err may be NULL


@pytest.mark.parametrize("name", ["norm", "norm_grad"])
def test_the_root_of_eps_has_a_reciprocal(name):
    """A row of zeros is multiplied by 1 / sqrt(eps), which binary32 has to hold."""
    for eps in (1e-300, 1e-78, 0.99e-75):
        assert call(name, eps=eps)[0] == s.ARITHMETIC, eps
    for eps in (1e-75, 1e-12, 1.0, 1e300):
        assert no_context(*call(name, eps=eps)), eps


def test_header_constants():
    text = (s.LIB_PATH.parents[1] / "include" / "pbsample.h").read_text()
    for name in ("HIDDEN_MAX_ROWS", "HIDDEN_MAX_COLS"):
        assert f"#define PB_{name} {getattr(hidden, name)}u" in text


class _Context:
    _ctx, device = 1, 0


class _Fake:
    """A buffer of another framework, on no device that it names."""

    def __init__(self, t):
        self.t, self.shape, self.dtype = t, t.shape, t.dtype

    def stride(self, i):
        return self.t.stride(i)

    def is_contiguous(self):
        return self.t.is_contiguous()

    def element_size(self):
        return self.t.element_size()

    def data_ptr(self):
        return self.t.data_ptr()


@pytest.fixture
def rows(monkeypatch):
    """HiddenRows whose library notes its calls."""
    made = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: made.append((name, a)) or 0

    monkeypatch.setattr(hidden, "lib", lambda: Lib())
    o = hidden.HiddenRows(sampler=_Context())
    o.made = made
    return o


def f(*shape, dtype=torch.float32):
    return _Fake(torch.zeros(shape, dtype=dtype))


def test_shapes_and_types_are_checked(rows):
    b = torch.int8
    q, w = f(3, 8, dtype=b), f(5, 8, dtype=b)
    rows.matmul(q, f(3), w, f(5), out=f(3, 5))
    for bad in (lambda: rows.matmul(f(3, 8), f(3), w, f(5), out=f(3, 5)),
                lambda: rows.matmul(q, f(2), w, f(5), out=f(3, 5)), lambda: rows.matmul(q, f(3), w, f(4), out=f(3, 5)),
                lambda: rows.matmul(q, f(3), f(5, 9, dtype=b), f(5), out=f(3, 5)),
                lambda: rows.matmul(q, f(3), w, f(5), out=f(3, 6)),
                lambda: rows.matmul(q, f(3), w, f(5), out=f(3, 5), bias=f(4)),
                lambda: rows.matmul(q, f(3), w, f(5), out=f(3, 5, dtype=torch.float64)),
                lambda: rows.matmul(_Fake(torch.zeros((8, 3), dtype=b).t()), f(3), w, f(5), out=f(3, 5)),
                lambda: rows.quantize(f(3, 8), q=f(3, 8), scale=f(3)),
                lambda: rows.quantize(f(3, 8), q=f(3, 7, dtype=b), scale=f(3)),
                lambda: rows.norm(f(3, 8), f(7), out=f(3, 8)), lambda: rows.norm(f(3, 8), f(1, 8), out=f(3, 8)),
                lambda: rows.norm(f(3, 8), f(8), residual=f(3, 9), out=f(3, 8)),
                lambda: rows.norm(f(3, 8), f(8), sum=f(3, 8, dtype=torch.bfloat16), out=f(3, 8)),
                lambda: rows.norm(f(3, 8), f(8), out=f(4, 8)),
                lambda: rows.norm_grad(f(3, 8), f(8), f(3, 8), grad_h=f(3, 8, dtype=torch.float16)),
                lambda: rows.norm_grad(f(3, 8), f(8), f(3, 8), grad_weight=f(7)),
                lambda: rows.norm_grad(f(3, 8), f(8), f(4, 8), grad_h=f(3, 8)),
                lambda: rows.embed(f(9, 8), f(3), out=f(3, 7)), lambda: rows.embed(f(9, 8), f(2), out=f(3, 8)),
                lambda: rows.embed(f(9, 8), f(3, dtype=torch.int64), out=f(3, 8)),
                lambda: rows.embed_grad(f(3, 8), f(3), table_grad=f(9, 7)),
                lambda: rows.embed(torch.zeros(9, 8), f(3), out=f(3, 8))):  # on the host
        with pytest.raises(ValueError):
            bad()
    assert [name for name, _ in rows.made] == ["pb_int8_matmul"]


def test_unsigned_bytes_are_no_8_bit_rows(rows):
    b = torch.int8
    for bad in (lambda: rows.matmul(f(3, 8, dtype=torch.uint8), f(3), f(5, 8, dtype=b), f(5), out=f(3, 5)),
                lambda: rows.matmul(f(3, 8, dtype=b), f(3), f(5, 8, dtype=torch.uint8), f(5), out=f(3, 5)),
                lambda: rows.quantize(f(3, 8), q=f(3, 8, dtype=torch.uint8), scale=f(3))):
        with pytest.raises(ValueError, match="signed bytes"):
            bad()
    assert not rows.made


def test_reservations_grow_by_doubling_and_cover_every_pair(rows):
    for n in range(1, 3000):
        rows._ensure(n, 896)
    rows.reserve(10, 5000)
    rows._ensure(2999, 5000)
    asked = [a[1:3] for name, a in rows.made]
    assert len(asked) <= 14 and asked[-1][0] >= 2999 and asked[-1][1] == 5000
    rows.norm_grad(f(4, 8), f(8), f(4, 8), grad_h=f(4, 8))  # needs no workspace
    rows._ensure(hidden.HIDDEN_MAX_ROWS, hidden.HIDDEN_MAX_COLS)
    assert rows._reserved == (hidden.HIDDEN_MAX_ROWS, hidden.HIDDEN_MAX_COLS)


def test_a_closed_context_refuses(rows):
    call = rows.bind_quantize(f(3, 8), q=f(3, 8, dtype=torch.int8), scale=f(3))
    call()
    rows.close()
    for bad in (call, lambda: rows.reserve(1, 1), lambda: rows.quantize(f(3, 8), q=f(3, 8, dtype=torch.int8), scale=f(3))):
        with pytest.raises(ValueError, match="closed"):
            bad()


# ---- the formulas ----

def test_gradients_against_differences():
    """The reference's gradients, which the kernels are held to, are those of the reference's outputs."""
    g = torch.Generator().manual_seed(3)
    rows, cols, eps = 4, 6, 1e-2

    def rand(*shape):
        return torch.randn(shape, generator=g, dtype=torch.float64)

    h, w, grad, more = rand(rows, cols), rand(cols), rand(rows, cols), rand(rows, cols)

    def loss(hv, wv):
        return ((ref.norm(hv, wv, eps) * grad).sum() + (hv * more).sum()).item()

    dh, dw = ref.norm_grad(h, w, grad, eps, more)
    step = 1e-6
    for i in range(rows):
        for j in range(cols):
            up, down = h.clone(), h.clone()
            up[i, j] += step
            down[i, j] -= step
            assert abs((loss(up, w) - loss(down, w)) / (2 * step) - dh[i, j]) < 1e-8
    for j in range(cols):
        up, down = w.clone(), w.clone()
        up[j] += step
        down[j] -= step
        assert abs((loss(h, up) - loss(h, down)) / (2 * step) - dw[j]) < 1e-8
    token = torch.tensor([2, -1, 0, 2])
    table = rand(3, cols)

    def looked_up(t):
        return (ref.embed(t, token, 1.7) * grad).sum().item()

    got, _ = ref.embed_grad(grad, token, 3, 1.7)
    for v in range(3):
        for j in range(cols):
            up, down = table.clone(), table.clone()
            up[v, j] += step
            down[v, j] -= step
            assert abs((looked_up(up) - looked_up(down)) / (2 * step) - got[v, j]) < 1e-8


def test_the_oracle_of_8_bit_rows_by_fractions():
    """Nearest whole numbers, halves to even ones, by whole-number arithmetic."""
    from fractions import Fraction

    g = torch.Generator().manual_seed(1)
    h = torch.randn((5, 40), generator=g)
    h[1] = torch.arange(-20, 20) / 2.0 + 0.5
    h[1, 0], h[2] = 127.0, 0.0
    w = torch.randn(40, generator=g)
    for weight in (None, w):
        q, top = ref.quantized(h, weight)
        for r in range(5):
            p = [Fraction(v) for v in h[r].tolist()]
            if weight is not None:
                p = [a * Fraction(b) for a, b in zip(p, w.tolist())]
            m = max(abs(v) for v in p)
            assert float(m) == top[r].item()
            assert q[r].tolist() == [round(127 * v / m) if m else 0 for v in p]  # Python rounds halves to even
    assert isinstance(np.longdouble(1) + 1, np.longdouble) and np.finfo(np.longdouble).nmant >= 63
