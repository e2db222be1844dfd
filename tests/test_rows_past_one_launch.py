"""More rows than a launch of one dimension holds (2^32 - 1 work items) are
refused, not run in part, by the entry points that have one.  Without a GPU:
nothing is launched."""

import ctypes

import pytest

import graspo_amd
from _capi import I32, I64, SZ, VP, SamplerParams, lib

F32 = ctypes.c_float
UNSUPPORTED = 2
P = 4096


def entry(name, *types):
    f = getattr(ctypes.CDLL(graspo_amd.LIB_PATH), name)
    f.argtypes, f.restype = types, I32
    return f


@pytest.mark.parametrize("N", [1 << 24, (1 << 24) + 1, 1 << 30])
def test_rows_of_256_threads(N):
    f = entry("gtp_lse_partial_rows", VP, I32, I64, I64, I64, I64, VP, I32, VP, I32, VP)
    assert f(P, 0, N, 8, 8, 0, P, 1, P, 0, None) == UNSUPPORTED
    f = entry("gtp_logprob_backward_rows", VP, I32, I64, I64, I64, I64, VP, I32, VP, VP, VP, I64,
              VP)
    assert f(P, 0, N, 8, 8, 0, P, 1, P, P, P, 8, None) == UNSUPPORTED
    f = entry("gtp_logprob_backward_split_rows", VP, I64, I64, I64, I64, VP, I32, VP, VP, VP, VP,
              I64, VP)
    assert f(P, N, 8, 8, 0, P, 1, P, P, P, P, 8, None) == UNSUPPORTED
    f = entry("gtp_graspo_loss_forward", VP, VP, VP, VP, I32, I64, I64, F32, F32, VP, VP, VP, VP)
    assert f(P, P, P, None, 0, N, 1, 0.8, 1.2, P, P, P, None) == UNSUPPORTED


@pytest.mark.parametrize("B,T", [(1 << 24, 1 << 8), (1, 1 << 32), (3, 1431655766)])
def test_positions_of_the_loss(B, T):
    f = entry("gtp_graspo_loss_backward", VP, VP, VP, VP, I32, VP, VP, I64, I64, F32, F32, VP, VP)
    assert f(P, P, P, None, 0, P, P, B, T, 0.8, 1.2, P, None) == UNSUPPORTED


@pytest.mark.parametrize("B", [1 << 22, (1 << 22) + 1, 1 << 30])
def test_rows_of_1024_threads(B):
    L = lib()
    for params in (SamplerParams(0.0, 0, 1.0, 1.0), SamplerParams(1.0, 0, 0.9, 1.0),
                   SamplerParams(1.0, 200, 1.0, 1.1)):
        args = [P, 1, B, 64, 64, None, 0, 0, None, 0, P, ctypes.byref(params), None, 0, *[P] * 7]
        assert L.gtp_sample_rows(*args, None, 0, None) == UNSUPPORTED
        assert L.gtp_sample_rows_noalloc(*args, None) == UNSUPPORTED
        r = ctypes.c_int32(0)
        assert L.gtp_sample_route(1, B, 64, 1, 0, 0, ctypes.byref(params), 0, ctypes.byref(r),
                                  None) == UNSUPPORTED
    f = entry("gtp_stream_read_rows", VP, I64, I64, I64, VP, VP)
    assert f(P, B, 16, 16, P, None) == UNSUPPORTED


def test_rows_of_the_matrix_products():
    f = entry("gtp_lm_head_logprob_rows", VP, I64, I64, I64, VP, I64, I64, VP, I32, VP, VP, VP, VP,
              VP, SZ, VP)
    rc = f(P, (1 << 26) + 1, 128, 128, P, 64, 128, P, 1, P, P, P, P, P, 1 << 60, None)
    assert rc == UNSUPPORTED
