"""Calls without a context are refused, each behind its other checks (no GPU)."""
import ctypes
import pathlib
import subprocess
import sys

import pytest

from promptboot_amd import sampler as s

A = [(1 << 50) + k * (1 << 40) for k in range(12)]  # addresses that nobody reads
V = s.VOCAB


def head_call(name, bytes_of):
    packed = getattr(s.lib(), bytes_of)(V, 64)
    if name == "decode":
        return (None, A[0], packed, V, 64, A[1], 3, A[2], 8, A[3], A[4], A[5], A[6], A[7], None, None, None, None)
    return (None, A[0], packed, V, 64, A[1], 3, A[2], 8, A[3], A[4], A[5], None, None, None, None)


CALLS = {
    "pb_context_reserve": lambda: (None, 5, 64),
    "pb_decode_step": lambda: (None, A[0], V, V, 3, A[1], 8, A[2], A[3], A[4], A[5], A[6], None, None, None),
    "pb_sample_batch": lambda: (None, A[0], V, V, 3, None, 0, None, A[1], A[2], None, None, None),
    "pb_lmhead_sample_batch": lambda: head_call("sample", "pb_lmhead_packed_bytes"),
    "pb_lmhead_q8_sample_batch": lambda: head_call("sample", "pb_lmhead_q8_packed_bytes"),
    "pb_lmhead_decode_step": lambda: head_call("decode", "pb_lmhead_packed_bytes"),
    "pb_lmhead_q8_decode_step": lambda: head_call("decode", "pb_lmhead_q8_packed_bytes"),
}


def refused(name):
    """(status, its record's status, its record's `needed`) of a call without a context."""
    e = s._Error()
    args = CALLS[name]()
    fn = getattr(s.lib(), name)
    assert len(args) + 1 == len(fn.argtypes), (name, len(args), len(fn.argtypes))
    return fn(*args, ctypes.byref(e)), e.status, e.needed


@pytest.mark.parametrize("name", CALLS)
def test_a_call_without_a_context_is_refused(name):
    # in a process of its own: one that is not refused ends it
    code = f"from tests.test_null_context import refused; print(*refused({name!r}))"
    done = subprocess.run([sys.executable, "-c", code], cwd=pathlib.Path(__file__).parents[1], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-500:]
    assert done.stdout.split() == [str(s.STATE), str(s.STATE), "1"]


def test_a_plan_without_a_context_is_no_call():
    code = "from promptboot_amd import sampler as s; s.lib().pb_context_set_segments(None, 4)"
    assert subprocess.run([sys.executable, "-c", code], cwd=pathlib.Path(__file__).parents[1]).returncode == 0
