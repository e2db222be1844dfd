"""What the look at states ahead of their move says, at the C ABI, without a
GPU: the same as the move itself would."""

import ctypes

import pytest

import graspo_amd
from test_beam_search_refusals import I64, INVALID, OK, UNSUPPORTED, VP, Shape, I32


def shape(run=64, row=256, sizes=(4, 1, 1, 1), strides=(64, 0, 0, 0)):
    return Shape(run, row, (I64 * 4)(*sizes), (I64 * 4)(*strides))


@pytest.mark.parametrize("code,change", [
    (OK, {}), (OK, dict(count=0, tensors=None)), (OK, dict(groups=0)), (OK, dict(beams=64)),
    (OK, dict(s=dict(run=0))),
    (INVALID, dict(count=-1)), (INVALID, dict(groups=-1)), (INVALID, dict(beams=0)),
    (INVALID, dict(tensors=None)), (INVALID, dict(tensors=(4096, None))),
    (INVALID, dict(s=dict(sizes=(0, 1, 1, 1)))), (INVALID, dict(s=dict(run=-1))),
    (UNSUPPORTED, dict(beams=65)), (UNSUPPORTED, dict(groups=1 << 31)),
    # an odd number of bytes past 2^31, by the row or by its address
    (UNSUPPORTED, dict(s=dict(run=(1 << 31) + 1))),
    (OK, dict(s=dict(run=1 << 31))),
    (UNSUPPORTED, dict(s=dict(run=1 << 31), tensors=(4096, 4097))),
    (UNSUPPORTED, dict(s=dict(run=1 << 31, row=(1 << 33) + 1))),
    (UNSUPPORTED, dict(s=dict(sizes=(1 << 31, 1, 1, 1)))),
])
def test_check(code, change):
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    L.gtp_reorder_states_check.argtypes = [VP, I64, ctypes.POINTER(Shape), I64, I32]
    a = dict(dict(tensors=(4096, 8192), count=2, groups=2, beams=3, s={}), **change)
    p = a["tensors"] and (VP * 2)(*a["tensors"])
    s = shape(**a["s"])
    assert L.gtp_reorder_states_check(p, a["count"], s, a["groups"], a["beams"]) == code
    assert L.gtp_reorder_states_check(p, 2, None, 2, 3) == INVALID
    if code != OK:  # refused before anything is launched
        L.gtp_reorder_states.argtypes = [VP, I64, ctypes.POINTER(Shape), VP, I64, I32, VP, VP]
        got = L.gtp_reorder_states(p, a["count"], s, 4096, a["groups"], a["beams"], None, None)
        assert got == code
