"""Operators on hidden-state rows at the sizes where one kernel's work ends and another's begins, and on both sides of
every choice between them, against the same in 64 bits.  Tolerances: tests/hidden_reference.py."""
import math

import pytest
import torch

from promptboot_amd import hip
from promptboot_amd.hidden import HIDDEN_MAX_ROWS, HiddenRows
from promptboot_amd.scores import SCORE_MAX_VOCAB
from tests import hidden_reference as ref
from tests.test_gpu_hidden import DEV, EPS, TYPES, gen, in_8_bits, make, make_bytes, near, space, untouched

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    o = HiddenRows(0)
    yield o
    o.close()


# ---- products ----

# rows x channels x columns, the columns in whole pieces of 16 bytes; run as they are and in rows that start anywhere
SIZES = [
    # few rows: both numbers of rows and of channels at which they end
    (1, 16_384, 64), (1, 16_385, 64), (2, 20_000, 48), (3, 20_000, 48), (16, 4_096, 32), (16, 4_097, 32), (17, 4_096, 48),
    (16, 16_385, 32), (17, 300, 32), (16, 1, 16), (7, 5, 4_096),
    # tiles of 32 x 32 with the contraction in eight, up to 256 and 512 of them
    (32, 8_192, 272), (32, 8_224, 272), (100, 2_040, 2_064), (32, 16_384, 144), (32, 16_416, 144), (64, 64, 1_040),
    # of 32 x 64 with the contraction in four, up to 256 and 512 of them
    (64, 16_384, 528), (64, 16_400, 528), (65, 5_440, 400), (65, 5_504, 400), (33, 16_384, 80), (33, 16_448, 80),
    # of 64 x 64 with the contraction in four, up to 256 of them
    (96, 8_192, 912), (1_000, 1_000, 272), (128, 8_192, 16), (128, 8_200, 272),
    # of 64 x 128 with the contraction in two
    (256, 8_192, 528), (200, 6_000, 400), (65, 8_200, 16),
    # of 64 x 128
    (300, 8_200, 144), (500, 8_190, 384), (20, 70_001, 80), (64, 40_000, 16),
    # of 128 x 256: one a workgroup, two and three; one step of columns and a ragged last one
    (1_024, 8_192, 272), (333, 30_001, 208), (129, 70_000, 16), (300, 50_001, 112), (3_000, 8_190, 128), (700, 6_150, 400),
    # of 256 x 256: one a workgroup, two and three; one step of columns, two and a ragged last one
    (1_000, 10_000, 896), (2_048, 16_384, 16), (2_000, 17_001, 112), (2_000, 17_001, 128), (1_990, 17_001, 208),
    (2_048, 16_400, 256), (1_024, 16_384, 288), (2_000, 20_000, 400),
]


@pytest.mark.parametrize("rows,channels,cols", SIZES)
def test_matmul(ops, rows, channels, cols):
    g = gen(rows + channels + cols)
    scale = torch.rand(rows, generator=g, device=DEV) * 1e-3
    weight_scale = torch.rand(channels, generator=g, device=DEV) * 1e-2
    for k, dtype in enumerate(("f32", "f16", "bf16")):
        # the outputs' rows in whole lines, in whole chunks and anywhere
        for pad, shift, out_pad in ((0, 0, -channels % 64), (16, 16, 8), (k + 1, 3, k)):
            q = make_bytes(g, rows, cols, pad, shift, lowest=-128)
            weight = make_bytes(g, channels, cols, pad, shift, lowest=-128)
            q[-1], weight[-1] = -128, -128  # the largest sums
            bias = torch.randn(channels, generator=g, device=DEV) if k != 1 else None
            full = space(rows, channels, TYPES[dtype], out_pad, shift, 5.0)
            ops.matmul(q, scale, weight, weight_scale, out=full[:, :channels], bias=bias)
            want, product = ref.matmul(q, scale, weight, weight_scale, bias)
            near(full[:, :channels], want, ref.matmul_tolerance(want, product, TYPES[dtype]), (dtype, pad, shift))
            assert untouched(full, channels, 5.0)


@pytest.mark.parametrize("rows", range(1, 18))
def test_matmul_of_few_rows(ops, rows):
    for cols in (1, 3, 15, 16, 17, 31, 63, 64, 65, 255, 257, 1_025):
        g = gen(rows * cols)
        for shift in (0, 1, 8):
            q, weight = make_bytes(g, rows, cols, shift, shift), make_bytes(g, 37, cols, shift, shift)
            scale, weight_scale = torch.rand(rows, generator=g, device=DEV), torch.rand(37, generator=g, device=DEV)
            full = space(rows, 37, torch.float32, 1, shift, 5.0)
            ops.matmul(q, scale, weight, weight_scale, out=full[:, :37])
            want, product = ref.matmul(q, scale, weight, weight_scale)
            near(full[:, :37], want, ref.matmul_tolerance(want, product, torch.float32), (cols, shift))
            assert untouched(full, 37, 5.0)


@pytest.mark.parametrize("rows,channels,cols", [(3, 50, 64), (20, 200, 48), (20, 200, 47), (70, 9_000, 64), (700, 6_150, 400),
                                                (2_000, 17_001, 112), (333, 30_001, 201)])
def test_zeros_keep_their_sign_without_a_bias(ops, rows, channels, cols):
    q, weight = torch.zeros((rows, cols), dtype=torch.int8, device=DEV), make_bytes(gen(1), channels, cols)
    scale, weight_scale = torch.full((rows,), -2.0, device=DEV), torch.ones(channels, device=DEV)
    weight_scale[1::2] = -1.0
    out = torch.full((rows, channels), 5.0, device=DEV)
    ops.matmul(q, scale, weight, weight_scale, out=out)
    want = torch.zeros(channels, device=DEV)
    want[0::2] = -0.0
    assert torch.equal(out.view(torch.int32), want.view(torch.int32).expand(rows, -1))
    ops.matmul(q, scale, weight, weight_scale, out=out, bias=torch.zeros(channels, device=DEV))
    assert not out.view(torch.int32).any()  # -0 + 0


# ---- the table's gradient ----

def table_gradient(ops, g, rows, vocab, cols, dtype, table_dtype, token, pad, shift=0):
    grad = make(g, rows, cols, dtype, pad=pad, shift=shift)
    total, absolute = ref.embed_grad(grad, token, vocab, 0.01)
    tol = ref.embed_grad_tolerance(total, total, absolute, 0.01, TYPES[table_dtype])
    full = space(vocab, cols, TYPES[table_dtype], pad=pad, shift=shift, fill=5.0)
    ops.embed_grad(grad, token.int(), table_grad=full[:, :cols], scale=0.01)
    near(full[:, :cols], total, tol, "dense")
    assert untouched(full, cols, 5.0)
    first = full.clone()
    ops.embed_grad(grad, token.int(), table_grad=full[:, :cols], scale=0.01)
    assert torch.equal(first, full)
    full[:, :cols] = 2.0
    ops.embed_grad(grad, token.int(), table_grad=full[:, :cols], scale=0.01, accumulate=True)
    near(full[:, :cols], total + 2.0, ref.embed_grad_tolerance(total, total + 2.0, absolute, 0.01, TYPES[table_dtype]), "added")
    assert untouched(full, cols, 5.0)


@pytest.mark.parametrize("rows", [1_023, 1_024, 1_025, 16_383, 16_384, 16_385, 20_481])
@pytest.mark.parametrize("vocab", [1, 511, 512, 513, 262_145])
def test_table_gradient_where_the_sort_changes(ops, rows, vocab):
    """One workgroup sorts up to 16,384 rows; ids take a pass for every 9 bits."""
    g = gen(rows + vocab)
    token = torch.randint(-1, vocab, (rows,), generator=g, device=DEV)
    token[0], token[-1], token[rows // 2] = vocab - 1, 0, vocab
    dtype = ["f32", "f16", "bf16"][rows % 3]
    table_gradient(ops, g, rows, vocab, 17, dtype, ["bf16", "f32", "f16"][vocab % 3], token, pad=rows % 2)


@pytest.mark.parametrize("run", [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 255, 257, 495, 496, 497, 511, 512, 513, 527, 528,
                                 529, 543, 544, 545, 560, 561, 1_040])
@pytest.mark.parametrize("first", [0, 1, 8, 15])
def test_table_gradient_of_runs(ops, run, first):
    """Equal tokens from any row of a part of 16 to any of another, short, just over 32 parts and longer."""
    g = gen(run)
    vocab = 9
    counts = [first, run, 3, run, 16, 1, run + 1]  # of the tokens 1, 2, ... as they are sorted
    token = torch.cat([torch.full((n,), i + 1, device=DEV) for i, n in enumerate(counts)])
    token = token[torch.randperm(token.numel(), generator=g, device=DEV)]
    for cols, pad in ((256, 0), (300, 3), (65, 1)):
        table_gradient(ops, g, token.numel(), vocab, cols, "f32", "f32", token, pad, shift=pad)


# ---- norms ----

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [1, 40, 513, 1_500, 4_097])
def test_8_bit_rows_at_the_borders_of_the_short_rounding(ops, dtype, cols):
    """Rows of a type with a weight of the same are rounded from binary32 products while the largest lies between 2^-60
    and 2^120; beside those and outside them, and rows of zeros among them."""
    t = TYPES[dtype]
    g = gen(cols)
    powers = [-130, -70, -61, -60, -59, -30, 0, 20, 60, 118, 119, 120, 121, 126] if dtype != "f16" else [-24, -14, -8, 0, 8, 14]
    for weight_power in ([-66, -60, -3, 0, 1, 60, 100] if dtype != "f16" else [-14, 0, 14]):
        x = torch.rand((len(powers) + 1, cols), generator=g, device=DEV, dtype=torch.float64) * 2 - 1
        x = torch.cat([(x[i] * 2.0 ** p)[None] for i, p in enumerate(powers)] + [x[-1:] * 0]).to(t)
        x = torch.where(x.isfinite(), x, torch.ones_like(x))
        w = ((0.5 + torch.rand(cols, generator=g, device=DEV, dtype=torch.float64)) * 2.0 ** weight_power).to(t)
        for weight in (w, w.float(), None):
            q = torch.full((len(x), cols + 1), 77, dtype=torch.int8, device=DEV)
            scale = torch.empty(len(x), device=DEV)
            ops.norm(x, weight, eps=EPS, q=q[:, :cols], scale=scale)
            want, top = ref.quantized(x, weight)
            # a scale past binary32 fails its row; one near its end may
            f = x.double()
            exact = top.to(DEV) / 127 / torch.sqrt((f * f).mean(1) + EPS)
            most = torch.finfo(torch.float32).max
            fails = scale.isnan()
            assert (exact[fails] > most * (1 - 4 * ref.E)).all() and (exact[~fails] < most * (1 + 4 * ref.E)).all()
            assert torch.equal(q[:, :cols].cpu(), torch.where(fails.cpu()[:, None], torch.zeros_like(want), want))
            near(scale[~fails], exact[~fails], ref.E * 1.001 * exact[~fails] + ref.tiny(torch.float32), "scale")
            assert (q[:, cols] == 77).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [511, 512, 513, 1_024, 1_025, 2_048, 2_049, 4_096, 4_097, 8_192, 8_193, 16_384, 16_385])
def test_norm_widths(ops, dtype, cols):
    """On both sides of every width at which more threads take a row, with the types equal and mixed."""
    for weight_dtype, grad_dtype in ((dtype, dtype), ("f16", "f32"), (None, dtype), (None, "f16")):
        g = gen(cols)
        rows = 5
        w = None
        if weight_dtype:
            w = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[weight_dtype])
        for pad in (0, 8, 1):
            x, residual = make(g, rows, cols, dtype, pad, pad), make(g, rows, cols, dtype, pad, pad)
            h = ref.rows_of(x, residual)
            out = space(rows, cols, TYPES[dtype], pad, pad, 5.0)
            q, scale = torch.full((rows, cols + pad), 77, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
            ops.norm(x, w, eps=EPS, residual=residual, out=out[:, :cols], q=q[:, :cols], scale=scale)
            want = ref.norm(h, w, EPS)
            near(out[:, :cols], want, ref.norm_tolerance(want, TYPES[dtype], w), "out")
            in_8_bits(q[:, :cols], scale, h, w, EPS, cols)
            grad = make(g, rows, cols, grad_dtype, pad, pad)
            dh, dw = space(rows, cols, TYPES[dtype], pad, pad, 5.0), torch.full((cols,), math.nan, device=DEV)
            ops.norm_grad(h, w, grad, eps=EPS, grad_h=dh[:, :cols], grad_weight=dw)
            want, want_weight = ref.norm_grad(h, w, grad, EPS)
            tol, tol_weight = ref.norm_grad_tolerances(h, w, grad, EPS, want, want_weight, TYPES[dtype])
            near(dh[:, :cols], want, tol, "grad_h")
            near(dw, want_weight, tol_weight, "grad_weight")
            assert untouched(out, cols, 5.0) and untouched(dh, cols, 5.0) and untouched(q, cols, 77)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("eps", [1e-75, 1e-30, 1e300])
def test_rows_of_zeros_with_any_eps(ops, dtype, eps):
    rows, cols = 3, 700
    x, w = torch.zeros((rows, cols), dtype=TYPES[dtype], device=DEV), torch.ones(cols, dtype=TYPES[dtype], device=DEV)
    out, q = torch.full((rows, cols), 5.0, device=DEV), torch.full((rows, cols), 77, dtype=torch.int8, device=DEV)
    scale, dw = torch.full((rows,), 5.0, device=DEV), torch.full((cols,), 5.0, device=DEV)
    ops.norm(x, w, eps=eps, out=out, q=q, scale=scale)
    assert (out == 0).all() and (q == 0).all() and (scale == 0).all()
    grad, dh = torch.full((rows, cols), 0.5, dtype=TYPES[dtype], device=DEV), torch.empty_like(x)
    ops.norm_grad(x, w, grad, eps=eps, grad_h=dh, grad_weight=dw)
    want = torch.full((rows, cols), 0.5 / math.sqrt(eps), dtype=torch.float64, device=DEV)
    if dtype == "f16" and eps < 1:  # past its largest
        assert dh.isinf().all()
    else:
        near(dh, want, ref.out_tolerance(want, TYPES[dtype], 2.01 * ref.E * want.abs()), "grad_h")
    assert (dw == 0).all()


# ---- the largest numbers of rows, ids and channels ----

def test_the_most_rows_and_channels(ops):
    g = gen(1)
    most = HIDDEN_MAX_ROWS
    q, scale = make_bytes(g, most, 16), torch.rand(most, generator=g, device=DEV)
    weight, weight_scale = make_bytes(g, 3, 16), torch.rand(3, generator=g, device=DEV)
    for cols in (16, 15):  # whole pieces and not
        out = torch.empty((most, 3), device=DEV)
        ops.matmul(q[:, :cols], scale, weight[:, :cols], weight_scale, out=out)
        want, product = ref.matmul(q[:, :cols], scale, weight[:, :cols], weight_scale)
        near(out, want, ref.matmul_tolerance(want, product, torch.float32), "rows")
    channels = SCORE_MAX_VOCAB
    weight, weight_scale = make_bytes(g, channels, 16), torch.rand(channels, generator=g, device=DEV)
    for rows in (1, 5, 20):
        for cols in (16, 15):
            out = torch.empty((rows, channels), dtype=torch.bfloat16, device=DEV)
            ops.matmul(q[:rows, :cols], scale[:rows], weight[:, :cols], weight_scale, out=out)
            for at in range(0, channels, 1 << 21):
                w, ws, o = weight[at:at + (1 << 21), :cols], weight_scale[at:at + (1 << 21)], out[:, at:at + (1 << 21)]
                want, product = ref.matmul(q[:rows, :cols], scale[:rows], w, ws)
                near(o, want, ref.matmul_tolerance(want, product, torch.bfloat16), (rows, cols, at))


@pytest.mark.parametrize("accumulate", [False, True])
def test_the_most_rows_and_ids_of_a_table(ops, accumulate):
    g = gen(2)
    rows, vocab, cols = HIDDEN_MAX_ROWS, SCORE_MAX_VOCAB, 3
    table = torch.randn((vocab, cols), generator=g, device=DEV)
    token = torch.randint(-1, vocab, (rows,), generator=g, device=DEV)
    token[:40_000] = vocab - 1
    out = torch.empty((rows, cols), device=DEV)
    ops.embed(table, token.int(), out=out)
    assert torch.equal(out, torch.where((token >= 0)[:, None], table[token.clamp(min=0)], torch.zeros_like(out)))
    grad = torch.randn((rows, cols), generator=g, device=DEV)
    total, absolute = ref.embed_grad(grad, token, vocab, 1.0)
    got = table.clone()
    ops.embed_grad(grad, token.int(), table_grad=got, accumulate=accumulate)
    want = total + table.double() if accumulate else total
    near(got, want, ref.embed_grad_tolerance(total, want, absolute, 1.0, torch.float32), "table")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_most_rows_of_a_norm(ops, dtype):
    g = gen(3)
    rows, cols = HIDDEN_MAX_ROWS, 9
    x, w = make(g, rows, cols, dtype), (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[dtype])
    out, q, scale = torch.empty_like(x), torch.empty((rows, cols), dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    ops.norm(x, w, eps=EPS, out=out, q=q, scale=scale)
    want = ref.norm(x, w, EPS)
    near(out, want, ref.norm_tolerance(want, TYPES[dtype], w), "out")
    in_8_bits(q, scale, x, w, EPS, cols)
    grad, dh, dw = make(g, rows, cols, dtype), torch.empty_like(x), torch.empty(cols, device=DEV)
    ops.norm_grad(x, w, grad, eps=EPS, grad_h=dh, grad_weight=dw)
    want, want_weight = ref.norm_grad(x, w, grad, EPS)
    tol, tol_weight = ref.norm_grad_tolerances(x, w, grad, EPS, want, want_weight, TYPES[dtype])
    near(dh, want, tol, "grad_h")
    near(dw, want_weight, tol_weight, "grad_weight")


@pytest.mark.parametrize("rows,cols", [(5_000, 1_500), (3_000, 520), (2_000, 1_025), (900, 5_000)])
def test_a_reservation_holds_for_every_smaller_call(rows, cols):
    """Narrower rows may be split over more workgroups than wider ones."""
    o = HiddenRows(0)
    try:
        o.reserve(rows, cols)
        for c in [c for c in (8, 511, 512, 513, 1_000, 1_024, 1_025, 1_500, 2_048, 4_096, cols) if c <= cols]:
            for r in (1, rows // 2, rows):
                x, dw = torch.ones((r, c), device=DEV), torch.empty(c, device=DEV)
                o.norm_grad(x, None, x, eps=EPS, grad_weight=dw)
                table, token = torch.empty((9, c), device=DEV), torch.full((r,), 3, dtype=torch.int32, device=DEV)
                o.embed_grad(x, token, table_grad=table)
                assert (table[3] == r).all() and (table[4] == 0).all()
                near(dw, torch.full((c,), r / math.sqrt(1 + EPS), dtype=torch.float64, device=DEV),
                     torch.full((c,), ref.E * 30.0 * r, device=DEV), "grad_weight")
        assert o._reserved == (rows, cols)
    finally:
        o.close()


# ---- captured ----

@pytest.mark.parametrize("rows", [700, 16_384, 16_385])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradients_in_a_captured_graph(rows, accumulate):
    g = gen(rows)
    vocab, cols = 3_000, 100
    ops = HiddenRows(0)
    try:
        ops.reserve(rows, cols)
        grad, token = make(g, rows, cols, "f32"), torch.zeros(rows, dtype=torch.int32, device=DEV)
        table = torch.zeros((vocab, cols), device=DEV)
        w, dh, dw = torch.ones(cols, device=DEV), torch.empty((rows, cols), device=DEV), torch.zeros(cols, device=DEV)
        want, want_weight = torch.empty_like(table), torch.empty_like(dw)
        stream = hip.Stream()

        def run(to, to_weight):
            ops.embed_grad(grad, token, table_grad=to, accumulate=accumulate, stream=stream)
            ops.norm_grad(grad, w, grad, grad_h=dh, grad_weight=to_weight, accumulate=accumulate, stream=stream)

        torch.cuda.synchronize()
        graph = hip.Graph(stream)
        graph.begin()
        run(table, dw)
        graph.end()
        for turn in range(4):
            grad.copy_(torch.randn((rows, cols), generator=g, device=DEV))
            token.copy_(torch.randint(-1, [1, vocab, 40, 2][turn], (rows,), generator=g, device=DEV))
            table.fill_(turn)
            dw.fill_(turn)
            want.copy_(table)
            want_weight.copy_(dw)
            torch.cuda.synchronize()
            graph.launch()
            stream.synchronize()
            got_dh = dh.clone()
            torch.cuda.synchronize()
            run(want, want_weight)
            stream.synchronize()
            assert torch.equal(table, want) and torch.equal(dw, want_weight) and torch.equal(dh, got_dh)
            total, absolute = ref.embed_grad(grad, token.long(), vocab, 1.0)
            base = float(turn) if accumulate else 0.0
            near(table, total + base, ref.embed_grad_tolerance(total, total + base, absolute, 1.0, torch.float32), turn)
        graph.close()
    finally:
        ops.close()


@pytest.mark.parametrize("rows,channels,cols", [(2, 5_000, 896), (30, 2_000, 512), (60, 9_000, 256), (100, 9_000, 256),
                                                (300, 9_000, 256), (700, 6_150, 400), (2_000, 17_001, 112), (50, 3_000, 201),
                                                (333, 30_001, 201)])
def test_products_in_a_captured_graph_and_on_two_streams(ops, rows, channels, cols):
    """A product of each kernel, replayed on new rows, and two of them at once."""
    g = gen(rows)
    q, weight = make_bytes(g, rows, cols), make_bytes(g, channels, cols)
    scale, weight_scale = torch.rand(rows, generator=g, device=DEV), torch.rand(channels, generator=g, device=DEV)
    out, other = torch.empty((rows, channels), device=DEV), torch.empty((rows, channels), device=DEV)
    streams = hip.Stream(), hip.Stream()
    calls = [ops.bind_matmul(q, scale, weight, weight_scale, out=o, stream=s) for o, s in zip((out, other), streams)]
    torch.cuda.synchronize()
    graph = hip.Graph(streams[0])
    graph.begin()
    calls[0]()
    calls[0]()
    graph.end()
    for _ in range(3):
        q.copy_(torch.randint(-127, 128, (rows, cols), generator=g, device=DEV))
        want, product = ref.matmul(q, scale, weight, weight_scale)
        out.fill_(5.0)
        other.fill_(5.0)
        torch.cuda.synchronize()
        graph.launch()
        for _ in range(3):
            calls[1]()
        for s in streams:
            s.synchronize()
        near(out, want, ref.matmul_tolerance(want, product, torch.float32), "replayed")
        assert torch.equal(out, other)
    graph.close()
