"""Scores and losses of logits rows, with their gradients, over libpbsample.so.

`RowScorer` reaches pb_token_logprobs, pb_token_logprobs_grad (in their _wide
forms), pb_top_logits, pb_distill_loss, pb_policy_loss and pb_preference_loss
(include/pbsample.h has their formulas, their row errors and which rows they skip).

Logits are device buffers [rows, columns] of binary32, binary16 or bfloat16:
tensors of another framework that shares this process's HIP runtime (their
rows may be strided), or `promptboot_amd.hip.DeviceArray`; 32-bit words count
as binary32 bit patterns, and 16-bit words need `dtype`.  The first `vocab`
columns (default: all) are the vocabulary.  Ids are 32-bit words with NO_TOKEN
(-1 in a signed buffer) for a row without a token; per-row inputs and outputs
are binary32, `err` [rows, 12] words (ERROR_DTYPE).  Gradients have the logits'
type and may be the logits themselves.

Every method checks its arguments, enqueues on `stream` and returns; each has a
`bind_` form that checks them once and returns a callable enqueuing that exact
call (it keeps the buffers and the stream alive), for loops over fixed buffers.
"""
from __future__ import annotations

import ctypes

from . import hip
from . import sampler as _s
from .sampler import OK, InferenceError, _check, _Error, _shape, lib, vp

F32, F16, BF16 = 0, 1, 2  # pb_dtype
SCORE_MAX_ROWS = 1_048_576
SCORE_MAX_VOCAB = 4_194_304
TOP_LOGITS_MAX = 128

_BY_NAME = {"float32": F32, "uint32": F32, "int32": F32, "float16": F16, "half": F16,
            "bfloat16": BF16, "f32": F32, "f16": F16, "bf16": BF16}


def _dtype_of(x, dtype) -> int:
    name = str(x.dtype if dtype is None else dtype).replace("torch.", "")
    if name not in _BY_NAME:
        raise ValueError(f"logits of type {name} are not supported (f32, f16 or bf16)")
    code = _BY_NAME[name]
    if _s._itemsize(x) != (4 if code == F32 else 2):
        raise ValueError(f"{name} logits do not have {_s._itemsize(x)}-byte elements")
    return code


def _on_device(x, name: str, device: int) -> None:
    """Refuses an array object that says it lies anywhere but on `device`."""
    where = getattr(x, "device", None)
    kind = getattr(where, "type", None)
    if kind is None:
        return
    index = getattr(where, "index", None)
    if kind != "cuda" or (index is not None and index != device):
        raise ValueError(f"{name} lies on {where}, the context on GPU {device}")


def _matrix(x, name: str, device: int):
    """(pointer, rows, columns, elements from one row to the next) of a 2-d buffer."""
    _on_device(x, name, device)
    shape = _shape(x)
    if len(shape) != 2:
        raise ValueError(f"{name} must have 2 dimensions, has shape {shape}")
    rows, columns = shape
    ld = columns
    if hasattr(x, "stride") and rows and columns:
        down, across = (int(x.stride(i)) for i in (0, 1))
        if columns > 1 and across != 1:
            raise ValueError(f"{name}: a row's elements must be next to each other")
        ld = columns if rows == 1 else down
        if ld < columns:
            raise ValueError(f"{name}: rows must not overlap")
    return vp(x.data_ptr()), rows, columns, ld


class RowScorer:
    """Scores and losses of logits rows on one GPU.

    Uses the context of `sampler` (a BatchSampler) when given, else one of its
    own on `device`.  The context's workspace is reserved before any call that
    needs more, so the enqueued calls never allocate; calls on one context
    must be ordered (one stream, or streams that the caller orders)."""

    def __init__(self, device: int = -1, sampler: "_s.BatchSampler | None" = None):
        self._own = sampler is None
        self.sampler = sampler if sampler is not None else _s.BatchSampler(device)
        self.device = self.sampler.device
        self._reserved = (0, 0)

    def _dev(self, x, name, **kw):
        _on_device(x, name, self.device)
        return _s._dev(x, name, **kw)

    def close(self) -> None:
        if self._own and self.sampler is not None:
            self.sampler.close()
        self.sampler = None

    def reserve(self, rows: int, vocab: int = _s.VOCAB) -> None:
        """Sizes the context for calls of up to `rows` rows of up to `vocab`
        ids, each at least as large as reserved before; a set-up call, it may
        allocate."""
        rows, vocab = max(rows, self._reserved[0]), max(vocab, self._reserved[1])
        e = _Error()
        _check(lib().pb_context_reserve_scores(self.sampler._ctx, rows, vocab, ctypes.byref(e)), e)
        self._reserved = (rows, vocab)

    def _ensure(self, rows: int, vocab: int) -> None:
        # An outgrown workspace stays allocated with the context (a captured graph may
        # use it): growing by doubling, all of them together are less than twice the last.
        def grown(need, have, most):
            return have if need <= have else max(need, min(2 * have, most))

        have = self._reserved
        if rows > have[0] or vocab > have[1]:
            self.reserve(grown(rows, have[0], SCORE_MAX_ROWS),
                         grown(vocab, have[1], SCORE_MAX_VOCAB))

    def _rows(self, logits, vocab, dtype):
        """The leading arguments of a call on `logits`, its rows, vocabulary and type."""
        if self.sampler is None:
            raise ValueError("the scorer's context is closed")
        ptr, rows, columns, ld = _matrix(logits, "logits", self.device)
        vocab = columns if vocab is None else int(vocab)
        if not 0 < vocab <= columns:
            raise ValueError(f"a vocabulary of {vocab} ids does not lie in {columns} columns")
        code = _dtype_of(logits, dtype)
        self._ensure(rows, vocab)
        return (self.sampler._ctx, ptr, code, vocab, ld, rows), rows, vocab, code

    def _grad(self, grad, rows, vocab, code, dtype):
        if grad is None:
            return None, 0
        ptr, grad_rows, columns, ld = _matrix(grad, "grad", self.device)
        if grad_rows != rows or columns < vocab:
            raise ValueError(f"grad has shape {_shape(grad)}, the logits {rows} rows of {vocab}")
        if _dtype_of(grad, dtype) != code:
            raise ValueError("grad must have the logits' type")
        return ptr, ld

    def _call(self, name: str, argv: tuple, keep: tuple):
        fn = getattr(lib(), name)

        def call():
            if self.sampler is None or not self.sampler._ctx:
                raise ValueError("the scorer's context is closed")
            e = _Error()
            st = fn(*argv, ctypes.byref(e))
            if st != OK:
                raise InferenceError(e)

        call.buffers = keep
        return call

    # ---- the calls ----

    def bind_token_logprobs(self, logits, token, *, logprob, lse=None, lse_low=None, entropy=None,
                            err=None, temperature: float = 1.0, vocab=None, dtype=None,
                            stream=None):
        head, rows, vocab, code = self._rows(logits, vocab, dtype)
        a = dict(rows=rows)
        argv = (*head, float(temperature), self._dev(token, "token", **a),
                self._dev(logprob, "logprob", **a), self._dev(lse, "lse", **a),
                self._dev(lse_low, "lse_low", **a),
                self._dev(entropy, "entropy", **a), self._dev(err, "err", row_elems=12, **a),
                vp(hip.stream_handle(stream)))
        return self._call("pb_token_logprobs_wide", argv,
                          (self, stream, logits, token, logprob, lse, lse_low, entropy, err))

    def token_logprobs(self, logits, token, **kw) -> None:
        """ln softmax(logits / temperature)[token] of each row; optionally the
        rows' log-sum-exp, what binary32 leaves out of it (lse_low, for the
        gradient) and entropy."""
        self.bind_token_logprobs(logits, token, **kw)()

    def bind_token_logprobs_grad(self, logits, token, lse, *, grad, lse_low=None,
                                 grad_logprob=None, grad_entropy=None, entropy=None,
                                 temperature: float = 1.0, vocab=None, dtype=None, stream=None):
        head, rows, vocab, code = self._rows(logits, vocab, dtype)
        a = dict(rows=rows)
        argv = (*head, float(temperature), self._dev(token, "token", **a),
                self._dev(lse, "lse", **a), self._dev(lse_low, "lse_low", **a),
                self._dev(entropy, "entropy", **a),
                self._dev(grad_logprob, "grad_logprob", **a),
                self._dev(grad_entropy, "grad_entropy", **a),
                *self._grad(grad, rows, vocab, code, dtype), vp(hip.stream_handle(stream)))
        return self._call("pb_token_logprobs_wide_grad", argv,
                          (self, stream, logits, token, lse, lse_low, entropy, grad_logprob,
                           grad_entropy, grad))

    def token_logprobs_grad(self, logits, token, lse, **kw) -> None:
        """The gradient of sum(grad_logprob * logprob + grad_entropy * entropy)
        by the logits, from the lse (and entropy) that token_logprobs left.  With
        lse_low too, 32-bit gradients are as exact as their type: lse alone is
        rounded, by up to 5e-7 of every q where it is 10."""
        self.bind_token_logprobs_grad(logits, token, lse, **kw)()

    def bind_top_logits(self, logits, k: int, *, token, value, lse=None, err=None,
                        temperature: float = 1.0, vocab=None, dtype=None, stream=None):
        head, rows, vocab, code = self._rows(logits, vocab, dtype)
        a = dict(rows=rows)
        argv = (*head, int(k), float(temperature), self._dev(token, "token", row_elems=k, **a),
                self._dev(value, "value", row_elems=k, **a), self._dev(lse, "lse", **a),
                self._dev(err, "err", row_elems=12, **a), vp(hip.stream_handle(stream)))
        return self._call("pb_top_logits", argv, (self, stream, logits, token, value, lse, err))

    def top_logits(self, logits, k: int, **kw) -> None:
        """Each row's k largest logits (a teacher's record): ids and raw values
        [rows, k], largest first, the lowest id first among equal ones."""
        self.bind_top_logits(logits, k, **kw)()

    def bind_distill_loss(self, logits, teacher_id, teacher_logit, *, loss, teacher_lse=None,
                          weight=None, lse=None, grad=None, err=None, temperature: float = 1.0,
                          vocab=None, dtype=None, stream=None):
        head, rows, vocab, code = self._rows(logits, vocab, dtype)
        shape = _shape(teacher_id)
        if len(shape) != 2 or _shape(teacher_logit) != shape or shape[0] != rows:
            raise ValueError(f"teacher_id and teacher_logit must be [{rows}, k], are {shape} and "
                             f"{_shape(teacher_logit)}")
        a = dict(rows=rows)
        argv = (*head, float(temperature), shape[1], self._dev(teacher_id, "teacher_id"),
                self._dev(teacher_logit, "teacher_logit"),
                self._dev(teacher_lse, "teacher_lse", **a), self._dev(weight, "weight", **a),
                self._dev(loss, "loss", **a), self._dev(lse, "lse", **a),
                *self._grad(grad, rows, vocab, code, dtype),
                self._dev(err, "err", row_elems=12, **a),
                vp(hip.stream_handle(stream)))
        return self._call("pb_distill_loss", argv,
                          (self, stream, logits, teacher_id, teacher_logit, teacher_lse, weight,
                           loss, lse, grad, err))

    def distill_loss(self, logits, teacher_id, teacher_logit, **kw) -> None:
        """Divergence of each row from a teacher's top logits, and weight times
        its gradient; with teacher_lse the teacher's remaining mass counts as
        one bucket, without it the listed ids are the whole teacher."""
        self.bind_distill_loss(logits, teacher_id, teacher_logit, **kw)()

    def bind_policy_loss(self, logits, token, old_logprob, advantage, *, loss, ref_logprob=None,
                         weight=None, clip_low: float = 0.2, clip_high: float = 0.2,
                         kl_coef: float = 0.0, logprob=None, kl=None, grad=None, err=None,
                         temperature: float = 1.0, vocab=None, dtype=None, stream=None):
        head, rows, vocab, code = self._rows(logits, vocab, dtype)
        a = dict(rows=rows)
        argv = (*head, float(temperature), self._dev(token, "token", **a),
                self._dev(old_logprob, "old_logprob", **a), self._dev(advantage, "advantage", **a),
                self._dev(ref_logprob, "ref_logprob", **a), self._dev(weight, "weight", **a),
                float(clip_low), float(clip_high), float(kl_coef), self._dev(loss, "loss", **a),
                self._dev(logprob, "logprob", **a), self._dev(kl, "kl", **a),
                *self._grad(grad, rows, vocab, code, dtype),
                self._dev(err, "err", row_elems=12, **a),
                vp(hip.stream_handle(stream)))
        return self._call("pb_policy_loss", argv,
                          (self, stream, logits, token, old_logprob, advantage, ref_logprob,
                           weight, loss, logprob, kl, grad, err))

    def policy_loss(self, logits, token, old_logprob, advantage, **kw) -> None:
        """Clipped policy loss with a KL term of each row, and weight times its
        gradient."""
        self.bind_policy_loss(logits, token, old_logprob, advantage, **kw)()

    def bind_preference_loss(self, logits, token, seq_start, *, loss, beta: float,
                             label_smoothing: float = 0.0, ref_logprob=None, weight=None,
                             logprob=None, grad=None, err=None, temperature: float = 1.0,
                             vocab=None, dtype=None, stream=None):
        head, rows, vocab, code = self._rows(logits, vocab, dtype)
        shape = _shape(seq_start)
        if len(shape) != 1 or shape[0] % 2 == 0:
            raise ValueError(f"seq_start must hold 2 x pairs + 1 offsets, has shape {shape}")
        pairs = shape[0] // 2
        one, two = dict(rows=pairs), dict(rows=2 * pairs)
        argv = (*head, float(temperature), self._dev(token, "token", rows=rows),
                self._dev(seq_start, "seq_start"), pairs,
                self._dev(ref_logprob, "ref_logprob", **two),
                self._dev(weight, "weight", **one), float(beta), float(label_smoothing),
                self._dev(loss, "loss", **one), self._dev(logprob, "logprob", **two),
                *self._grad(grad, rows, vocab, code, dtype),
                self._dev(err, "err", row_elems=12, **one),
                vp(hip.stream_handle(stream)))
        return self._call("pb_preference_loss", argv,
                          (self, stream, logits, token, seq_start, ref_logprob, weight, loss,
                           logprob, grad, err))

    def preference_loss(self, logits, token, seq_start, **kw) -> None:
        """Loss of pairs of sequences (rows seq_start[s] .. seq_start[s + 1];
        2i chosen, 2i + 1 rejected) by their paired log ratios, and weight times
        its gradient."""
        self.bind_preference_loss(logits, token, seq_start, **kw)()
