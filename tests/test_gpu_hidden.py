"""Operators on hidden-state rows against the same in 64 bits, at the sizes, strides, types and values where they
could go wrong.  Tolerances: tests/hidden_reference.py."""
import math

import numpy as np
import pytest
import torch

from promptboot_amd import sampler as s
from promptboot_amd.hidden import HiddenRows
from tests import hidden_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    o = HiddenRows(0)
    yield o
    o.close()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def space(rows, cols, dtype, pad=0, shift=0, fill=math.nan):
    """Rows of `cols` + `pad` elements that start `shift` elements into their allocation, all of it `fill`."""
    flat = torch.full((rows * (cols + pad) + shift + 8,), fill, dtype=dtype, device=DEV)
    return flat[shift:shift + rows * (cols + pad)].view(rows, cols + pad)


def make(g, rows, cols, dtype, pad=0, shift=0, spread=1.0):
    x = space(rows, cols, TYPES[dtype], pad, shift)[:, :cols]
    x.copy_(torch.randn((rows, cols), generator=g, device=DEV) * spread)
    return x


def make_bytes(g, rows, cols, pad=0, shift=0, lowest=-127):
    x = space(rows, cols, torch.int8, pad, shift, fill=77)[:, :cols]
    x.copy_(torch.randint(lowest, 128, (rows, cols), generator=g, device=DEV))
    return x


def records(rows):
    return torch.full((rows, 12), 77, dtype=torch.int32, device=DEV)


def read_errors(err):
    torch.cuda.synchronize()
    return err.cpu().numpy().view(s.ERROR_DTYPE).reshape(-1)


def near(got, want, tol, what):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][:3].tolist(),
                           want[bad][:3].tolist(), (tol.expand_as(got)[bad][:3]).tolist())


def untouched(full, cols, fill):
    rest = full[:, cols:]
    return bool((rest.isnan() if math.isnan(fill) else rest == fill).all())


# ---- table rows ----

COLS = [1, 7, 8, 9, 63, 64, 65, 896, 1001, 2049, 5000]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_dtype", ["f32", "f16", "bf16"])
def test_embed_types_and_widths(ops, dtype, out_dtype):
    for k, cols in enumerate(COLS):
        g = gen(k)
        rows, vocab = [1, 3, 40, 260][k % 4], [1, 2, 300, 5000][k % 4]
        table = make(g, vocab, cols, dtype, pad=k % 3, shift=k % 5)
        token = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        if rows > 2:
            token[0], token[1], token[2] = -1, vocab, vocab - 1
        full = space(rows, cols, TYPES[out_dtype], pad=(k + 1) % 4, shift=k % 3, fill=5.0)
        err = records(rows)
        ops.embed(table, token.int(), out=full[:, :cols], scale=31.6, err=err)
        want = ref.embed(table, token, 31.6)
        near(full[:, :cols], want, ref.embed_tolerance(want, TYPES[out_dtype]), (cols, "out"))
        assert untouched(full, cols, 5.0)
        e = read_errors(err)
        for r in range(rows):
            if token[r] == vocab:
                assert (e[r]["status"], e[r]["position"], e[r]["needed"], e[r]["available"], e[r]["detail"]) == \
                    (s.TOKEN_ID, r, vocab, vocab, 2 << 32)
            else:
                assert not e[r:r + 1].view(np.uint8).any()
    # ids far past the table, as unsigned words
    token = torch.tensor([2**31 - 1, -2, -2**31], dtype=torch.int32, device=DEV)
    out = space(3, cols, TYPES[out_dtype], fill=5.0)
    ops.embed(table, token, out=out)
    assert out.isnan().all()


def test_a_scale_of_one_keeps_the_bits(ops):
    table = make(gen(1), 50, 100, "f32", spread=1e-39)  # below the normal range too
    token = torch.arange(50, device=DEV).int()
    out = space(50, 100, torch.float32)
    ops.embed(table, token, out=out)
    assert torch.equal(out.view(torch.int32), table.contiguous().view(torch.int32))


def tokens_like(kind, rows, vocab, g):
    if kind == "one":
        t = torch.full((rows,), vocab // 2, device=DEV)
    elif kind == "distinct":
        t = torch.randperm(max(rows, vocab), generator=g, device=DEV)[:rows] % vocab
    elif kind == "runs":
        t = (torch.arange(rows, device=DEV) // 33) % vocab
    else:  # frequent ones, as text has
        t = (vocab ** torch.rand(rows, generator=g, device=DEV, dtype=torch.float64)).long().clamp(max=vocab) - 1
    if rows > 4:
        t[torch.rand(rows, generator=g, device=DEV) < 0.2] = -1
        t[rows // 3] = vocab  # adds nothing
    return t


GRADS = [(1, 1, 1), (2, 3, 9), (31, 5, 64), (32, 5, 7), (33, 1, 896), (64, 40, 130), (65, 511, 513), (300, 512, 100),
         (1000, 513, 896), (4095, 70, 33), (4096, 3000, 64), (4097, 100, 520), (9000, 262_145, 9), (20_000, 1000, 300),
         (70_000, 50_257, 24)]


@pytest.mark.parametrize("kind", ["one", "distinct", "runs", "text"])
@pytest.mark.parametrize("rows,vocab,cols", GRADS)
def test_embed_grad(ops, rows, vocab, cols, kind):
    g = gen(rows + vocab)
    names = ["f32", "f16", "bf16"]
    dtype, table_dtype = names[(rows + cols) % 3], names[rows % 3]
    grad = make(g, rows, cols, dtype, pad=rows % 3, shift=cols % 4)
    token = tokens_like(kind, rows, vocab, g)
    dead = (token < 0) | (token >= vocab)
    grad[dead] = math.nan  # what such rows hold does not matter
    # half-precision sums of many rows stay in range
    scale = 1.0 if table_dtype != "f16" else 0.01
    total, absolute = ref.embed_grad(grad, token, vocab, scale)
    full = space(vocab, cols, TYPES[table_dtype], pad=vocab % 3, shift=vocab % 2, fill=5.0)
    ops.embed_grad(grad, token.int(), table_grad=full[:, :cols], scale=scale)
    near(full[:, :cols], total, ref.embed_grad_tolerance(total, total, absolute, scale, TYPES[table_dtype]), "dense")
    assert untouched(full, cols, 5.0)
    first = full.clone()
    ops.embed_grad(grad, token.int(), table_grad=full[:, :cols], scale=scale)
    assert torch.equal(first, full)  # sums repeat bit for bit
    # added to what is there; rows without a token keep their bits
    old = torch.randn((vocab, cols), generator=g, device=DEV).to(TYPES[table_dtype])
    full[:, :cols] = old
    ops.embed_grad(grad, token.int(), table_grad=full[:, :cols], scale=scale, accumulate=True)
    want = old.double() + total
    near(full[:, :cols], want, ref.embed_grad_tolerance(total, want, absolute, scale, TYPES[table_dtype]), "added")
    hit = torch.zeros(vocab, dtype=torch.bool, device=DEV)
    hit[token[~dead]] = True
    assert torch.equal(full[:, :cols][~hit], old[~hit]) and untouched(full, cols, 5.0)


def test_embed_grad_without_rows(ops):
    grad = torch.empty((0, 16), device=DEV)
    token = torch.empty(0, dtype=torch.int32, device=DEV)
    table = torch.full((9, 16), 3.0, device=DEV)
    ops.embed_grad(grad, token, table_grad=table, accumulate=True)
    assert (table == 3.0).all()
    ops.embed_grad(grad, token, table_grad=table)
    assert (table == 0.0).all()


@pytest.mark.parametrize("rows", [5, 100])
def test_embed_grad_of_masked_rows_only(ops, rows):
    grad = torch.full((rows, 40), math.nan, device=DEV)
    token = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    table = torch.full((20, 40), 3.0, device=DEV)
    ops.embed_grad(grad, token, table_grad=table, accumulate=True)
    assert (table == 3.0).all()
    ops.embed_grad(grad, token, table_grad=table)
    assert (table == 0.0).all()


# ---- norms ----

# rows x columns: a chunk's edges, each plan's edges
NORMS = [(1, 1), (3, 7), (2, 8), (5, 9), (7, 511), (4, 512), (3, 513), (70, 896), (9, 1023), (5, 1024), (6, 1025),
         (3, 2048), (4, 2049), (2, 4096), (3, 4097), (2, 8192), (3, 8193), (2, 16_384), (2, 16_385), (1, 32_767),
         (2, 32_768), (700, 130)]


def in_8_bits(q, scale, h, weight, eps, cols, norm=True):
    want_q, top = ref.quantized(h, weight)
    assert torch.equal(q.cpu(), want_q), (q.cpu() != want_q).nonzero()[:3].tolist()
    want = top.to(DEV) / 127.0
    if norm:
        f = h.double()
        want = want / torch.sqrt((f * f).mean(1) + eps)
    near(scale, want, ref.E * 1.001 * want + ref.tiny(torch.float32), "scale")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", NORMS)
def test_norm(ops, rows, cols, dtype):
    g = gen(rows * cols)
    weight_dtype = ["f32", dtype, None, "bf16"][cols % 4]
    out_dtype = [dtype, "f32", "f16"][rows % 3]
    weight = None
    if weight_dtype:
        weight = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[weight_dtype])
    x = make(g, rows, cols, dtype, pad=rows % 3, shift=cols % 3)
    residual = make(g, rows, cols, dtype, pad=1, spread=3.0) if rows % 2 else None
    h = ref.rows_of(x, residual)
    t = TYPES[dtype]
    total, out = space(rows, cols, t, 2, 1, 5.0), space(rows, cols, TYPES[out_dtype], 1, 3, 5.0)
    q = torch.full((rows, cols + 3), 77, dtype=torch.int8, device=DEV)
    scale = torch.full((rows,), math.nan, device=DEV)
    err = records(rows)
    ops.norm(x, weight, eps=EPS, residual=residual, sum=total[:, :cols], out=out[:, :cols], q=q[:, :cols], scale=scale,
             err=err)
    assert torch.equal(total[:, :cols], h)
    want = ref.norm(h, weight, EPS)
    near(out[:, :cols], want, ref.norm_tolerance(want, TYPES[out_dtype], weight), "out")
    in_8_bits(q[:, :cols], scale, h, weight, EPS, cols)
    assert untouched(total, cols, 5.0) and untouched(out, cols, 5.0) and untouched(q, cols, 77)
    assert not read_errors(err).view(np.uint8).any()
    # each output alone is the same
    out2, q2, scale2 = torch.empty_like(out), torch.empty_like(q), torch.empty_like(scale)
    ops.norm(x, weight, eps=EPS, residual=residual, out=out2[:, :cols])
    ops.norm(x, weight, eps=EPS, residual=residual, q=q2[:, :cols], scale=scale2)
    assert torch.equal(out2[:, :cols], out[:, :cols]) and torch.equal(q2[:, :cols], q[:, :cols])
    assert torch.equal(scale2, scale)
    # in the inputs' places
    x2, r2 = x.clone(), residual.clone() if residual is not None else None
    ops.norm(x2, weight, eps=EPS, residual=r2, sum=x2 if rows % 4 else r2, q=q2[:, :cols], scale=scale2)
    assert torch.equal(x2 if rows % 4 or r2 is None else r2, h) and torch.equal(q2[:, :cols], q[:, :cols])
    if out_dtype == dtype:
        x2 = x.clone()
        ops.norm(x2, weight, eps=EPS, residual=residual, out=x2)
        assert torch.equal(x2, out[:, :cols])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 9), (70, 896), (300, 1025), (3, 5000), (2, 20_000), (2, 32_768)])
def test_quantize(ops, rows, cols, dtype):
    g = gen(rows + cols)
    x = make(g, rows, cols, dtype, pad=3, shift=1, spread=0.02)
    x[rows // 2] = 0.0
    q = torch.full((rows, cols + 5), 77, dtype=torch.int8, device=DEV)
    scale, err = torch.full((rows,), math.nan, device=DEV), records(rows)
    ops.quantize(x, q=q[:, :cols], scale=scale, err=err)
    in_8_bits(q[:, :cols], scale, x, None, EPS, cols, norm=False)
    assert scale[rows // 2] == 0.0 and untouched(q, cols, 77)
    assert not read_errors(err).view(np.uint8).any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_halves_go_to_even_numbers(ops, dtype):
    """127 p / max is a half exactly for every odd multiple of max / 254; beside it, the nearest values decide."""
    t = TYPES[dtype]
    k = torch.arange(-127, 127, device=DEV)
    row = torch.cat([(2 * k + 1).double() / 2, torch.tensor([127.0], dtype=torch.float64, device=DEV)])
    rows = []
    for scale in (1.0, 0.25, 2.0 ** -10):  # exact in every type: 8 bits
        x = (row * scale).to(t)
        assert torch.equal(x.double(), row * scale)
        up, down = (torch.nextafter(x.float(), torch.full_like(x.float(), v)).to(t) for v in (math.inf, -math.inf))
        rows += [x, torch.cat([up[:-1], x[-1:]]), torch.cat([down[:-1], x[-1:]])]
    x = torch.stack(rows)
    q, scale = torch.empty(x.shape, dtype=torch.int8, device=DEV), torch.empty(len(rows), device=DEV)
    ops.quantize(x, q=q, scale=scale)
    want, _ = ref.quantized(x, None)
    assert torch.equal(q.cpu(), want)
    assert (q[0, :-1].cpu() % 2 == 0).all()
    # under a weight whose products need 48 bits: p = (2k + 1) / 2 w for one w is a tie, as before
    w = torch.full((row.numel(),), 1.0 + 2.0 ** -20, device=DEV)
    ops.norm(x, w, q=q, scale=scale)
    assert torch.equal(q.cpu(), ref.quantized(x, w)[0])
    w = 1.0 + torch.rand(row.numel(), generator=gen(3), device=DEV)
    ops.norm(x, w, q=q, scale=scale)
    assert torch.equal(q.cpu(), ref.quantized(x, w)[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [1e-44, 1e-38, 1e-30, 1e-12, 1e12, 1e30, 5e37])
@pytest.mark.parametrize("weight_spread", [1e-30, 1.0, 1e30])
def test_norms_of_very_small_and_large_rows(ops, dtype, spread, weight_spread):
    g = gen(5)
    rows, cols = 6, 777
    x = torch.randn((rows, cols), generator=g, device=DEV).double().mul(spread).to(TYPES[dtype])
    x[0] = 0.0
    w = (torch.rand(cols, generator=g, device=DEV) * weight_spread).to(TYPES[dtype])
    out, q = torch.empty((rows, cols), device=DEV), torch.empty((rows, cols), dtype=torch.int8, device=DEV)
    scale = torch.empty(rows, device=DEV)
    ops.norm(x, w, eps=EPS, out=out, q=q, scale=scale)
    want = ref.norm(x, w, EPS)
    f = x.double()
    rstd = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)
    # an rstd below the normal range is off by half of the smallest step
    tol = ref.norm_tolerance(want, torch.float32, w) + want.abs() * (ref.tiny(torch.float32) / rstd)
    near(out, want, tol, "out")
    want_q, top = ref.quantized(x, w)
    assert torch.equal(q.cpu(), want_q)
    want_scale = top.to(DEV) * rstd[:, 0] / 127
    near(scale, want_scale, 1.001 * ref.E * want_scale + ref.tiny(torch.float32), "scale")


@pytest.mark.parametrize("rows,cols", [(6, 100), (6, 3000), (6, 9000)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_that_are_not_finite_fail_alone(ops, rows, cols, dtype):
    g = gen(cols)
    x, residual = make(g, rows, cols, dtype), make(g, rows, cols, dtype)
    w = (1 + 0.1 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[dtype])
    x[1, cols - 1] = math.nan
    x[2, 40] = math.inf
    residual[2, 50] = -math.inf
    x[4, 3], residual[4, 3] = math.inf, -math.inf
    h = ref.rows_of(x, residual)
    for use in ("out", "q", "both"):
        out = torch.full((rows, cols), 5.0, dtype=TYPES[dtype], device=DEV)
        total, q = torch.empty_like(out), torch.full((rows, cols), 77, dtype=torch.int8, device=DEV)
        scale, err = torch.full((rows,), 5.0, device=DEV), records(rows)
        kw = {}
        if use != "q":
            kw.update(out=out)
        if use != "out":
            kw.update(q=q, scale=scale)
        ops.norm(x, w, eps=EPS, residual=residual, sum=total, err=err, **kw)
        e = read_errors(err)
        failed = {1: cols - 1, 2: 40, 4: 3}
        for r in range(rows):
            if r in failed:
                bits = h[r, failed[r]].float().view(torch.int32).item() & 0xFFFFFFFF
                got = (e[r]["status"], e[r]["position"], e[r]["available"], e[r]["detail"])
                assert got[:2] == (s.NONFINITE_INPUT, r) and got[3] == 7 << 32 | failed[r]
                if not h[r, failed[r]].isnan():
                    assert got[2] == bits
            else:
                assert not e[r:r + 1].view(np.uint8).any()
        ok = [0, 3, 5]
        assert torch.equal(total[ok], h[ok]) and torch.equal(total.isnan(), h.isnan())
        if use != "q":
            assert out[list(failed)].isnan().all()
            want = ref.norm(h[ok], w, EPS)
            near(out[ok], want, ref.norm_tolerance(want, TYPES[dtype], w), "out")
        if use != "out":
            assert scale[list(failed)].isnan().all() and (q[list(failed)] == 0).all()
            in_8_bits(q[ok], scale[ok], h[ok], w, EPS, cols)


def test_weights_that_are_not_finite_fail_the_8_bit_rows(ops):
    x = make(gen(1), 3, 900, "bf16")
    w = torch.ones(900, dtype=torch.bfloat16, device=DEV)
    w[77] = math.inf
    q, scale, err = torch.full((3, 900), 77, dtype=torch.int8, device=DEV), torch.empty(3, device=DEV), records(3)
    ops.norm(x, w, q=q, scale=scale, err=err)
    e = read_errors(err)
    assert scale.isnan().all() and (q == 0).all()
    assert (e["status"] == s.NONFINITE_INPUT).all() and (e["detail"] == 7 << 32 | 77).all()
    # products that binary32 does not hold, and a scale that it does not
    w = torch.full((900,), 3e38, dtype=torch.bfloat16, device=DEV)
    x[0], x[1] = 3e38, 1.0  # row 0: y = 3e38 everywhere, its products 9e76
    x[2] = 0.0
    x[2, 5] = 1.0  # y = 30 * 3e38
    ops.norm(x, w, q=q, scale=scale, err=err)
    e = read_errors(err)
    assert (q[:2] == 127).all() and scale[:2].isfinite().all() and (e["status"][:2] == s.OK).all()
    assert scale[2].isfinite() and (q[2].nonzero() == 5).all()  # 30 * 3e38 / 127
    x = torch.zeros((1, 32_768), dtype=torch.bfloat16, device=DEV)
    x[0, 9] = 1.0
    w = torch.full((32_768,), 3e38, dtype=torch.bfloat16, device=DEV)  # y = 181 * 3e38: over 127 * 3.4e38
    q, err = torch.full((1, 32_768), 77, dtype=torch.int8, device=DEV), records(1)
    ops.norm(x, w, q=q, scale=scale[:1], err=err)
    e = read_errors(err)
    assert scale[0].isnan() and (q == 0).all() and e["status"][0] == s.NONFINITE_INPUT
    assert e["detail"][0] == 7 << 32 | 32_768


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", NORMS + [(2049, 64), (5000, 33), (1030, 2100), (530, 9000)])
def test_norm_grad(ops, rows, cols, dtype):
    g = gen(rows + cols)
    weight_dtype = ["f32", dtype, None][cols % 3]
    grad_dtype = [dtype, "f32", "bf16"][rows % 3]
    weight = None
    if weight_dtype:
        weight = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[weight_dtype])
    h = make(g, rows, cols, dtype, pad=rows % 3, shift=cols % 3, spread=2.0)
    grad = make(g, rows, cols, grad_dtype, pad=1)
    more = make(g, rows, cols, dtype, pad=2) if rows % 2 else None
    want, want_weight = ref.norm_grad(h, weight, grad, EPS, more)
    tol, tol_weight = ref.norm_grad_tolerances(h, weight, grad, EPS, want, want_weight, TYPES[dtype])
    dh = space(rows, cols, TYPES[dtype], 1, 1, 5.0)
    dw = torch.full((cols + 2,), 5.0, device=DEV)
    ops.norm_grad(h, weight, grad, eps=EPS, grad_sum=more, grad_h=dh[:, :cols], grad_weight=dw[1:-1])
    near(dh[:, :cols], want, tol, "grad_h")
    near(dw[1:-1], want_weight, tol_weight, "grad_weight")
    assert untouched(dh, cols, 5.0) and dw[0] == 5.0 and dw[-1] == 5.0
    # each gradient alone is the same, and repeats; the weight's added to what is there
    dh2, dw2 = torch.empty_like(dh), torch.full((cols,), 7.0, device=DEV)
    ops.norm_grad(h, weight, grad, eps=EPS, grad_sum=more, grad_h=dh2[:, :cols])
    assert torch.equal(dh2[:, :cols], dh[:, :cols])
    ops.norm_grad(h, weight, grad, eps=EPS, grad_weight=dw2, accumulate=True)
    near(dw2, want_weight + 7.0, tol_weight + ref.E * 7.0, "added")
    ops.norm_grad(h, weight, grad, eps=EPS, grad_weight=dw2)
    assert torch.equal(dw2, dw[1:-1])
    # in the inputs' places
    places = [h] + ([grad] if grad_dtype == dtype else []) + ([more] if more is not None else [])
    for k in range(len(places)):
        a = [h.clone(), grad.clone(), more.clone() if more is not None else None]
        to = a[0] if places[k] is h else a[1] if places[k] is grad else a[2]
        ops.norm_grad(a[0], weight, a[1], eps=EPS, grad_sum=a[2], grad_h=to)
        assert torch.equal(to, dh[:, :cols])


def test_norm_grad_without_rows(ops):
    h = torch.empty((0, 16), device=DEV)
    dw = torch.full((16,), 3.0, device=DEV)
    ops.norm_grad(h, None, h, grad_weight=dw, accumulate=True)
    assert (dw == 3.0).all()
    ops.norm_grad(h, None, h, grad_weight=dw)
    assert (dw == 0.0).all()


# ---- products ----

PRODUCTS = [(1, 1, 1), (1, 16, 896), (1, 1000, 896), (2, 17, 15), (3, 64, 16), (5, 65, 17), (15, 257, 63), (16, 130, 64),
            (17, 64, 65), (31, 200, 127), (32, 96, 128), (33, 300, 129), (48, 1024, 2048), (63, 127, 896), (64, 128, 1001),
            (65, 129, 896), (100, 513, 4096), (128, 256, 640), (129, 255, 1000), (255, 1111, 96), (257, 700, 896),
            (300, 4099, 100), (1, 33, 32_768), (40, 70, 32_767), (130, 140, 20_001), (513, 1030, 257)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,channels,cols", PRODUCTS)
def test_matmul(ops, rows, channels, cols, dtype):
    g = gen(rows + channels + cols)
    for pad, shift in ((0, 0), (16 - cols % 16, 0), (rows % 5 + 1, cols % 7)):
        q = make_bytes(g, rows, cols, pad, shift, lowest=-128)
        weight = make_bytes(g, channels, cols, pad, (shift * 3) % 5, lowest=-128)
        q[0], weight[0] = -128, -128  # the largest sums
        scale = torch.rand(rows, generator=g, device=DEV) * 1e-3
        weight_scale = torch.rand(channels, generator=g, device=DEV) * 1e-2
        bias = torch.randn(channels, generator=g, device=DEV) if cols % 2 else None
        full = space(rows, channels, TYPES[dtype], pad, shift, 5.0)
        ops.matmul(q, scale, weight, weight_scale, out=full[:, :channels], bias=bias)
        want, product = ref.matmul(q, scale, weight, weight_scale, bias)
        near(full[:, :channels], want, ref.matmul_tolerance(want, product, TYPES[dtype]), (pad, shift))
        assert untouched(full, channels, 5.0)


def test_matmul_of_a_whole_vocabulary(ops):
    g = gen(7)
    q, weight = make_bytes(g, 70, 896), make_bytes(g, s.VOCAB, 896)
    scale, weight_scale = torch.rand(70, generator=g, device=DEV), torch.rand(s.VOCAB, generator=g, device=DEV)
    for rows in (1, 2, 33, 70):
        out = torch.empty((rows, s.VOCAB), device=DEV)
        ops.matmul(q[:rows], scale[:rows], weight, weight_scale, out=out)
        want, product = ref.matmul(q[:rows], scale[:rows], weight, weight_scale)
        near(out, want, ref.matmul_tolerance(want, product, torch.float32), rows)


@pytest.mark.parametrize("rows", [3, 70, 300])
def test_scales_that_are_not_finite_fail_their_row_or_channel(ops, rows):
    g = gen(rows)
    q, weight = make_bytes(g, rows, 200), make_bytes(g, 150, 200)
    scale, weight_scale = torch.ones(rows, device=DEV), torch.ones(150, device=DEV)
    scale[1], weight_scale[140] = math.nan, math.nan
    out = torch.empty((rows, 150), device=DEV)
    ops.matmul(q, scale, weight, weight_scale, out=out)
    bad = torch.zeros((rows, 150), dtype=torch.bool, device=DEV)
    bad[1], bad[:, 140] = True, True
    assert torch.equal(out.isnan(), bad)


def test_rows_past_32_bit_offsets(ops):
    """Buffers of over 4 GB: the last rows lie where a 32-bit offset does not reach."""
    g = gen(9)
    rows, cols = 70_000, 32_768
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn((3, cols), generator=g, device=DEV)
    token = torch.arange(rows, device=DEV).int()
    token[-1] = 5
    out = torch.empty((3, cols), dtype=torch.bfloat16, device=DEV)
    ops.embed(x, token[-3:].clamp(min=rows - 3), out=out)
    assert torch.equal(out[:2], x[-3:-1])
    q, scale = torch.full((rows, cols), 77, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    ops.quantize(x, q=q, scale=scale)
    in_8_bits(q[-3:], scale[-3:], x[-3:], None, EPS, cols, norm=False)
    assert (q[:100] == 0).all() and (scale[:-3] == 0).all()
    ops.norm(x, None, out=x)
    near(x[-3:-1], ref.norm(out[:2], None, 1e-6), ref.norm_tolerance(ref.norm(out[:2], None, 1e-6), x.dtype), "norm")
    w, ws = make_bytes(g, 4, cols), torch.ones(4, device=DEV)
    y = torch.empty((rows, 4), device=DEV)
    ops.matmul(q, scale, w, ws, out=y)
    want, product = ref.matmul(q[-3:], scale[-3:], w, ws)
    near(y[-3:], want, ref.matmul_tolerance(want, product, torch.float32), "rows")
    assert (y[:-3] == 0).all()
    y = torch.empty((4, rows), device=DEV)  # as channels
    ops.matmul(w, ws, q, scale, out=y)
    want, product = ref.matmul(w, ws, q[-3:], scale[-3:])
    near(y[:, -3:], want, ref.matmul_tolerance(want, product, torch.float32), "channels")
