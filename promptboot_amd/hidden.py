"""Hidden-state rows around a head, over libpbsample.so: table rows of tokens, norms, 8-bit rows, their products.

`HiddenRows` reaches pb_embed_rows, pb_embed_rows_grad, pb_norm_rows,
pb_norm_rows_grad, pb_quantize_rows and pb_int8_matmul (include/pbsample.h has their
formulas, and what becomes of rows without a token and of values that are not finite).

Rows are device buffers [rows, columns] of binary32, binary16 or bfloat16: tensors of
another framework that shares this process's HIP runtime (their rows may be strided), or
`promptboot_amd.hip.DeviceArray`; 32-bit words count as binary32 bit patterns, and
16-bit words need a type's name (`dtype` for the rows, `weight_dtype`, `out_dtype` and
the like for other buffers, which default to what the buffer says).  8-bit rows are
[rows, columns] of signed bytes.  Tokens are 32-bit words with NO_TOKEN (-1 in a signed
buffer) for a row without one; scales, biases and the weight's gradient are binary32,
`err` is [rows, 12] words (ERROR_DTYPE).

Every method checks its arguments, enqueues on `stream` and returns; each has a `bind_`
form that checks them once and returns a callable enqueuing that exact call (it keeps the
buffers and the stream alive), for loops over fixed buffers.  The callable's `check()`
raises what the library would refuse of the call, but for a missing reservation, and
enqueues nothing.
"""
from __future__ import annotations

import ctypes

from . import hip
from . import sampler as _s
from .sampler import OK, STATE, InferenceError, _check, _Error, _shape, lib, vp
from .scores import _dtype_of, _matrix, _on_device

HIDDEN_MAX_ROWS = 1_048_576
HIDDEN_MAX_COLS = 32_768


class HiddenRows:
    """Operators on hidden-state rows on one GPU.

    Uses the context of `sampler` (a BatchSampler) when given, else one of its own on
    `device`.  The context's workspace is reserved before any gradient that needs more
    (as much as that one needs; reserve() does it beforehand), so the enqueued calls never
    allocate; gradients on one context must be ordered (one stream, or streams that the
    caller orders)."""

    def __init__(self, device: int = -1, sampler: "_s.BatchSampler | None" = None):
        self._own = sampler is None
        self.sampler = sampler if sampler is not None else _s.BatchSampler(device)
        self.device = self.sampler.device
        self._reserved = (0, 0)

    def close(self) -> None:
        if self._own and self.sampler is not None:
            self.sampler.close()
        self.sampler = None

    def reserve(self, rows: int, cols: int) -> None:
        """Sizes the context for gradients of up to `rows` rows of up to `cols` columns, in
        every pair of these and of what was reserved before (a number that grows again
        doubles at least); a set-up call, it may allocate."""
        self._context()
        self._ensure(rows, cols)

    def _ensure(self, rows: int, cols: int) -> None:
        # An outgrown workspace stays allocated with the context (a captured graph may
        # use it): growing by doubling, all of them together are less than twice the last.
        def grown(need, have, most):
            return have if need <= have else max(need, min(2 * have, most))

        have = self._reserved
        if rows > have[0] or cols > have[1]:
            both = grown(rows, have[0], HIDDEN_MAX_ROWS), grown(cols, have[1], HIDDEN_MAX_COLS)
            self._reserve("pb_context_reserve_hidden", *both)
            self._reserved = both

    def _reserve(self, name: str, rows: int, cols: int) -> None:
        e = _Error()
        _check(getattr(lib(), name)(self._context(), rows, cols, ctypes.byref(e)), e)

    def workspace_bytes(self) -> int:
        """What the context holds for gradients."""
        return lib().pb_context_hidden_bytes(self._context())

    def _context(self):
        if self.sampler is None or not self.sampler._ctx:
            raise ValueError("the context is closed")
        return self.sampler._ctx

    def _dev(self, x, name, **kw):
        _on_device(x, name, self.device)
        return _s._dev(x, name, **kw)

    def _rows(self, x, name, dtype, rows=None, cols=None):
        """(pointer, type, distance of rows) of a buffer of `rows` rows of at least `cols` columns."""
        if x is None:
            return None, 0, 0
        ptr, r, c, ld = _matrix(x, name, self.device)
        if rows is not None and r != rows or cols is not None and c != cols:
            raise ValueError(f"{name} has shape {_shape(x)}, not ({rows}, {cols})")
        return ptr, _dtype_of(x, dtype), ld

    def _bytes(self, x, name, rows=None, cols=None):
        """(pointer, distance of rows) of 8-bit rows."""
        if x is None:
            return None, 0
        ptr, r, c, ld = _matrix(x, name, self.device)
        kind = str(x.dtype).replace("torch.", "")
        if kind != "int8":
            raise ValueError(f"{name} must hold signed bytes, not {kind}")
        if rows is not None and r != rows or cols is not None and c != cols:
            raise ValueError(f"{name} has shape {_shape(x)}, not ({rows}, {cols})")
        return ptr, ld

    def _weight(self, x, name, dtype, cols):
        """(pointer, type) of a weight of `cols` elements."""
        if x is None:
            return None, 0
        _on_device(x, name, self.device)
        if _shape(x) != (cols,):
            raise ValueError(f"{name} has shape {_shape(x)}, not ({cols},)")
        return _s._dev(x, name, itemsize=_s._itemsize(x)), _dtype_of(x, dtype)

    def _call(self, name: str, argv: tuple, keep: tuple):
        fn = getattr(lib(), name)

        def call():
            self._context()
            e = _Error()
            st = fn(*argv, ctypes.byref(e))
            if st != OK:
                raise InferenceError(e)

        def check():
            # without a context the library checks everything else, and enqueues nothing
            self._context()
            e = _Error()
            st = fn(None, *argv[1:], ctypes.byref(e))
            if st != OK and not (st == STATE and e.needed == 1):
                raise InferenceError(e)

        call.buffers, call.check = keep, check
        return call

    # ---- the calls ----

    def bind_embed(self, table, token, *, out, scale: float = 1.0, err=None, dtype=None, out_dtype=None, stream=None):
        ctx = self._context()
        ptr, vocab, cols, ld = _matrix(table, "table", self.device)
        code = _dtype_of(table, dtype)
        rows = _shape(out)[0]
        po, out_code, out_ld = self._rows(out, "out", out_dtype, rows, cols)
        argv = (ctx, ptr, code, vocab, cols, ld, rows, self._dev(token, "token", rows=rows), float(scale), po, out_code,
                out_ld, self._dev(err, "err", rows=rows, row_elems=12), vp(hip.stream_handle(stream)))
        return self._call("pb_embed_rows", argv, (self, stream, table, token, out, err))

    def embed(self, table, token, **kw) -> None:
        """out[r] = scale * table[token[r]]: zeros for a row without a token, NaN (and a
        record) for an id that the table does not have."""
        self.bind_embed(table, token, **kw)()

    def bind_embed_grad(self, grad, token, *, table_grad, scale: float = 1.0, accumulate: bool = False, dtype=None,
                        table_dtype=None, stream=None):
        ctx = self._context()
        ptr, rows, cols, ld = _matrix(grad, "grad", self.device)
        code = _dtype_of(grad, dtype)
        vocab = _shape(table_grad)[0]
        pt, table_code, table_ld = self._rows(table_grad, "table_grad", table_dtype, vocab, cols)
        argv = (ctx, ptr, code, vocab, cols, ld, rows, self._dev(token, "token", rows=rows), float(scale),
                int(accumulate), pt, table_code, table_ld, vp(hip.stream_handle(stream)))
        self._reserve("pb_context_reserve_embed_grad", rows, cols)
        return self._call("pb_embed_rows_grad", argv, (self, stream, grad, token, table_grad))

    def embed_grad(self, grad, token, **kw) -> None:
        """The table's gradient: each token's rows of `grad` added up in their order, times
        `scale`; zeros elsewhere, or, with `accumulate`, added to what is there."""
        self.bind_embed_grad(grad, token, **kw)()

    def bind_norm(self, x, weight=None, *, eps: float = 1e-6, residual=None, sum=None, out=None, q=None, scale=None,
                  err=None, dtype=None, weight_dtype=None, out_dtype=None, stream=None):
        ctx = self._context()
        ptr, rows, cols, ld = _matrix(x, "x", self.device)
        code = _dtype_of(x, dtype)
        pr, res_code, res_ld = self._rows(residual, "residual", dtype, rows, cols)
        ps, sum_code, sum_ld = self._rows(sum, "sum", dtype, rows, cols)
        if residual is not None and res_code != code or sum is not None and sum_code != code:
            raise ValueError("residual and sum must have the rows' type")
        pw, weight_code = self._weight(weight, "weight", weight_dtype, cols)
        po, out_code, out_ld = self._rows(out, "out", out_dtype, rows, cols)
        pq, q_ld = self._bytes(q, "q", rows, cols)
        argv = (ctx, ptr, code, cols, ld, rows, pr, res_ld, pw, weight_code, float(eps), ps, sum_ld, po, out_code,
                out_ld, pq, q_ld, self._dev(scale, "scale", rows=rows),
                self._dev(err, "err", rows=rows, row_elems=12), vp(hip.stream_handle(stream)))
        return self._call("pb_norm_rows", argv, (self, stream, x, weight, residual, sum, out, q, scale, err))

    def norm(self, x, weight=None, **kw) -> None:
        """Root-mean-square norm of x (+ residual, the sum kept in `sum`): in `out`, and in 8
        bits in `q` with the rows' `scale`."""
        self.bind_norm(x, weight, **kw)()

    def bind_norm_grad(self, h, weight, grad, *, eps: float = 1e-6, grad_sum=None, grad_h=None, grad_weight=None,
                       accumulate: bool = False, dtype=None, weight_dtype=None, grad_dtype=None, stream=None):
        ctx = self._context()
        ptr, rows, cols, ld = _matrix(h, "h", self.device)
        code = _dtype_of(h, dtype)
        pg, grad_code, grad_ld = self._rows(grad, "grad", grad_dtype, rows, cols)
        ps, sum_code, sum_ld = self._rows(grad_sum, "grad_sum", dtype, rows, cols)
        ph, h_code, h_ld = self._rows(grad_h, "grad_h", dtype, rows, cols)
        if grad_sum is not None and sum_code != code or grad_h is not None and h_code != code:
            raise ValueError("grad_sum and grad_h must have the rows' type")
        pw, weight_code = self._weight(weight, "weight", weight_dtype, cols)
        argv = (ctx, ptr, code, cols, ld, rows, pw, weight_code, float(eps), pg, grad_code, grad_ld, ps, sum_ld, ph,
                h_ld, self._dev(grad_weight, "grad_weight", rows=cols), int(accumulate),
                vp(hip.stream_handle(stream)))
        if grad_weight is not None:
            self._reserve("pb_context_reserve_norm_grad", rows, cols)
        return self._call("pb_norm_rows_grad", argv,
                          (self, stream, h, weight, grad, grad_sum, grad_h, grad_weight))

    def norm_grad(self, h, weight, grad, **kw) -> None:
        """The norm's gradients from its rows h (norm's `sum`, or its x without a residual)
        and the gradient by its output: by h, with grad_sum added, and by the weight."""
        self.bind_norm_grad(h, weight, grad, **kw)()

    def bind_quantize(self, x, *, q, scale, err=None, dtype=None, stream=None):
        ctx = self._context()
        ptr, rows, cols, ld = _matrix(x, "x", self.device)
        code = _dtype_of(x, dtype)
        pq, q_ld = self._bytes(q, "q", rows, cols)
        argv = (ctx, ptr, code, cols, ld, rows, pq, q_ld, self._dev(scale, "scale", rows=rows),
                self._dev(err, "err", rows=rows, row_elems=12), vp(hip.stream_handle(stream)))
        return self._call("pb_quantize_rows", argv, (self, stream, x, q, scale, err))

    def quantize(self, x, **kw) -> None:
        """Rows in 8 bits with a scale each: weights (a channel a row) or activations."""
        self.bind_quantize(x, **kw)()

    def bind_matmul(self, q, scale, weight, weight_scale, *, out, bias=None, out_dtype=None, stream=None):
        ctx = self._context()
        ptr, rows, cols, ld = _matrix(q, "q", self.device)
        self._bytes(q, "q")
        channels = _shape(weight)[0]
        pw, weight_ld = self._bytes(weight, "weight", channels, cols)
        po, out_code, out_ld = self._rows(out, "out", out_dtype, rows, channels)
        argv = (ctx, ptr, ld, self._dev(scale, "scale", rows=rows), rows, cols, pw, weight_ld,
                self._dev(weight_scale, "weight_scale", rows=channels), channels,
                self._dev(bias, "bias", rows=channels), po, out_code, out_ld, vp(hip.stream_handle(stream)))
        return self._call("pb_int8_matmul", argv, (self, stream, q, scale, weight, weight_scale, bias, out))

    def matmul(self, q, scale, weight, weight_scale, **kw) -> None:
        """out[r][n] = scale[r] * weight_scale[n] * (q[r] . weight[n]) (+ bias[n]) of 8-bit
        rows and 8-bit channels; the dot products are exact."""
        self.bind_matmul(q, scale, weight, weight_scale, **kw)()
