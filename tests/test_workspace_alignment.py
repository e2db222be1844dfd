"""Workspaces that the training step's entry points cannot use as they lie, at
the C ABI: refused before anything is launched.  Without a GPU."""

import ctypes

import pytest

import graspo_amd
from test_linear_logprob_refusals import GOOD, INVALID, LinearRows

VP, I64, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
BIG = 1 << 40


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_linear(off):
    """Rows go straight to LDS from it, 16 bytes at a time."""
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    L.gtp_linear_logprob_rows.argtypes = [ctypes.POINTER(LinearRows), VP, VP, VP, VP, VP, VP, SZ, VP]
    L.gtp_linear_logprob_backward.argtypes = [ctypes.POINTER(LinearRows), VP, VP, VP, VP, VP, VP, SZ, VP]
    r = ctypes.byref(LinearRows(**GOOD))
    assert L.gtp_linear_logprob_rows(r, 4096, 4096, None, None, None, 4096 + off, BIG, None) == INVALID
    assert L.gtp_linear_logprob_backward(r, 4096, 4096, None, 4096, 4096, 4096 + off, BIG, None) == INVALID


@pytest.mark.parametrize("off", [1, 2, 4])
def test_norm(off):
    """64-bit sums."""
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    L.gtp_grad_norm.argtypes = [VP, VP, VP, I64, ctypes.c_int, VP, VP, SZ, VP]
    args = (VP * 1)(4096), (I64 * 1)(10), (ctypes.c_int32 * 1)(0), 1, 2, 4096
    assert L.gtp_grad_norm(*args, 4096 + off, 1 << 20, None) == INVALID
