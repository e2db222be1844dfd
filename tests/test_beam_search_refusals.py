"""Calls that the beam search and the states' moves refuse, without a GPU."""

import ctypes
import math

import pytest
import torch

import graspo_amd
from graspo_amd import decode_loop as dl
from graspo_amd.beam_search import (beam_finish, beam_start, beam_step, expand_states, length_of,
                                    reorder_states_)

VP, I64, I32, SZ, F64 = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t,
                         ctypes.c_double)
OK, INVALID, UNSUPPORTED = 0, 1, 2


class Rows(ctypes.Structure):
    _fields_ = [(n, VP) for n in ("logits", "allow_mask", "scores", "done")] + [
        (n, I64) for n in ("groups", "vocab", "group_stride", "beam_stride", "mask_stride")] + [
        (n, I32) for n in ("dtype", "beams", "candidates")]


class State(ctypes.Structure):
    _fields_ = [(n, VP) for n in (
        "scores", "pool_scores", "pool_rows", "pool_steps", "done", "out_tokens", "out_parents",
        "out_scores", "out_pool_scores", "out_pool_rows", "out_pool_steps", "out_done")] + [
        ("eos", I64), ("pad", I64), ("length", F64), ("step", I32), ("early", I32)]


class Shape(ctypes.Structure):
    _fields_ = [("run_bytes", I64), ("row_stride", I64), ("sizes", I64 * 4), ("strides", I64 * 4)]


def lib():
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    P = ctypes.POINTER
    L.gtp_beam_workspace_bytes.argtypes = [P(Rows)]
    L.gtp_beam_workspace_bytes.restype = SZ
    L.gtp_beam_candidates.argtypes = [P(Rows), VP, VP, VP, VP, VP, SZ, VP]
    L.gtp_beam_step.argtypes = [P(Rows), P(State), VP, VP, SZ, VP]
    L.gtp_beam_advance.argtypes = [VP, VP, VP, I64, I32, I32, P(State), VP]
    L.gtp_beam_finish.argtypes = [VP] * 7 + [I64, I32, I32, F64, I64, I64, I32, VP, VP, VP, I64, VP]
    L.gtp_reorder_states.argtypes = [VP, I64, P(Shape), VP, I64, I32, VP, VP]
    L.gtp_expand_states.argtypes = [VP, VP, I64, P(Shape), I64, I32, VP]
    return L


def rows(**change):
    a = dict(logits=4096, allow_mask=None, scores=4096, done=None, groups=2, vocab=1000,
             group_stride=4000, beam_stride=1000, mask_stride=32, dtype=1, beams=4, candidates=8)
    a.update(change)
    return Rows(**a)


def state(**change):
    a = {n: 4096 for n, t in State._fields_ if t is VP}
    a.update(eos=1, pad=0, length=1.0, step=0, early=0)
    a.update(change)
    return State(**a)


@pytest.mark.parametrize("change,code", [
    (dict(groups=-1), INVALID), (dict(beams=0), INVALID), (dict(candidates=0), INVALID),
    (dict(vocab=0), INVALID), (dict(dtype=3), INVALID), (dict(logits=None), INVALID),
    (dict(scores=None), INVALID), (dict(beam_stride=-1), INVALID), (dict(group_stride=-1), INVALID),
    (dict(logits=4097), INVALID), (dict(allow_mask=4096, mask_stride=31), INVALID),
    (dict(beams=33), UNSUPPORTED), (dict(candidates=65), UNSUPPORTED),
    (dict(vocab=(1 << 31) - 1), UNSUPPORTED), (dict(groups=1 << 23), UNSUPPORTED),
])
def test_beam_rows(change, code):
    L = lib()
    r = rows(**change)
    assert L.gtp_beam_candidates(r, 4096, 4096, 4096, 4096, 4096, 1 << 40, None) == code
    s = state(scores=r.scores or 4096)
    if r.scores:
        assert L.gtp_beam_step(r, s, 4096, 4096, 1 << 40, None) in (code, INVALID)


def test_beam_buffers():
    L = lib()
    r = rows()
    need = L.gtp_beam_workspace_bytes(r)
    assert need == 2 * 4 * 1 * 13 * 8  # one slice per row: 12 keys and a sum
    assert L.gtp_beam_workspace_bytes(rows(beams=40)) == 0
    for bad in ((None, 4096, 4096), (4096, None, 4096), (4096, 4096, None)):
        assert L.gtp_beam_candidates(r, *bad, None, 4096, need, None) == INVALID
    for ws, n in ((None, need), (4096, need - 1), (4100, need)):
        assert L.gtp_beam_candidates(r, 4096, 4096, 4096, None, ws, n, None) == INVALID
        assert L.gtp_beam_step(rows(done=4096), state(), None, ws, n, None) == INVALID
    assert L.gtp_beam_candidates(None, 4096, 4096, 4096, None, 4096, need, None) == INVALID
    assert L.gtp_beam_candidates(rows(groups=0), None, None, None, None, None, 0, None) == OK


@pytest.mark.parametrize("change", [dict(length=0.0), dict(length=-1.0), dict(length=math.nan),
                                    dict(length=math.inf), dict(step=-1)]
                         + [{n: None} for n, t in State._fields_ if t is VP])
def test_beam_state(change):
    L = lib()
    s = state(**change)
    assert L.gtp_beam_advance(4096, 4096, 4096, 2, 4, 8, s, None) == INVALID
    assert L.gtp_beam_step(rows(done=4096), s, None, 4096, 1 << 30, None) == INVALID


def test_beam_step_takes_the_states_scores():
    L = lib()
    assert L.gtp_beam_step(rows(done=4096, scores=8192), state(), None, 4096, 1 << 30, None) == INVALID
    assert L.gtp_beam_step(rows(), state(), None, 4096, 1 << 30, None) == INVALID
    assert L.gtp_beam_step(rows(done=4096), None, None, 4096, 1 << 30, None) == INVALID
    for a, code in (((-1, 4, 8), INVALID), ((2, 0, 8), INVALID), ((2, 4, 0), INVALID),
                    ((2, 33, 8), UNSUPPORTED), ((2, 4, 65), UNSUPPORTED), ((1 << 23, 4, 8), UNSUPPORTED)):
        assert L.gtp_beam_advance(4096, 4096, 4096, *a, state(), None) == code
    for bad in ((None, 4096, 4096), (4096, None, 4096), (4096, 4096, None)):
        assert L.gtp_beam_advance(*bad, 2, 4, 8, state(), None) == INVALID


def test_beam_finish_entry_point():
    L = lib()
    def call(p=(4096,) * 7, groups=2, beams=4, steps=5, length=1.0, give=2, out=(4096,) * 3, room=5):
        return L.gtp_beam_finish(*p, groups, beams, steps, length, 1, 0, give, *out, room, None)
    for bad in (dict(groups=-1), dict(beams=0), dict(steps=-1), dict(give=0), dict(give=5),
                dict(room=4), dict(length=0.0), dict(length=math.nan)):
        assert call(**bad) == INVALID
    for i in range(7):
        assert call(p=tuple(None if j == i else 4096 for j in range(7))) == INVALID
    for i in range(3):
        assert call(out=tuple(None if j == i else 4096 for j in range(3))) == INVALID
    assert call(beams=33, give=1) == UNSUPPORTED
    assert call(groups=0, p=(None,) * 7, out=(None,) * 3) == OK


def test_states_entry_points():
    L = lib()
    ptrs = (VP * 2)(4096, 8192)
    def shape(run=64, row=64, sizes=(1, 1, 1, 1), strides=(0, 0, 0, 0)):
        return Shape(run, row, (I64 * 4)(*sizes), (I64 * 4)(*strides))
    def both(p=ptrs, n=2, s=None, groups=2, beams=4, parents=4096):
        s = shape() if s is None else s
        a = L.gtp_reorder_states(p, n, s, parents, groups, beams, None, None)
        b = L.gtp_expand_states(p, p, n, s, groups, beams, None)
        assert a == b
        return a
    for bad in (dict(p=None), dict(n=-1), dict(groups=-1), dict(beams=0), dict(p=(VP * 2)(4096, None)),
                dict(s=shape(run=-1)), dict(s=shape(sizes=(1, 0, 1, 1)))):
        assert both(**bad) == INVALID
    for bad in (dict(beams=65), dict(groups=1 << 30), dict(s=shape(run=1 << 36)),
                dict(s=shape(sizes=(1 << 31, 1, 1, 1))), dict(s=shape(sizes=(1 << 20, 1 << 20, 1, 1))),
                dict(s=shape(run=16, sizes=(1 << 30, 2, 1, 1)))):
        assert both(**bad) == UNSUPPORTED
    assert L.gtp_reorder_states(ptrs, 2, None, 4096, 2, 4, None, None) == INVALID
    assert L.gtp_reorder_states(ptrs, 2, shape(), None, 2, 4, None, None) == INVALID
    assert L.gtp_expand_states(ptrs, None, 2, shape(), 2, 4, None) == INVALID
    assert both(n=0) == both(groups=0) == both(s=shape(run=0)) == OK


def test_python_arguments():
    st = beam_start(2, 3, "cpu")
    args = dict(eos_token_id=1, pad_token_id=0)
    x = torch.zeros(6, 50)
    for bad in (x.double(), x.int()):
        with pytest.raises(ValueError, match="float32"):
            beam_step(bad, st, **args)
    for bad in (x[:5], x[0], x.view(3, 2, 50), x[None, None]):
        with pytest.raises(ValueError, match="logits"):
            beam_step(bad, st, **args)
    for p in (1e6, -1e6, math.nan, math.inf):
        with pytest.raises(ValueError, match="length_penalty"):
            beam_step(x, st._replace(step=5), length_penalty=p, **args)
    assert length_of(1, 1e6) == 1.0 and length_of(4, 0.5) == 2.0
    for g, k in ((1, 0), (1, 33), (-1, 2)):
        with pytest.raises(ValueError, match="beams"):
            beam_start(g, k, "cpu")
    t, p = torch.zeros(4, 6, dtype=torch.int64), torch.zeros(4, 6, dtype=torch.int32)
    for n in (0, 4):
        with pytest.raises(ValueError, match="num_return"):
            beam_finish(st._replace(step=4), t, p, num_return=n, **args)
    for a, b in ((t[:3], p[:3]), (t, p[:, :5]), (t[:, :5], p[:, :5])):
        with pytest.raises(ValueError, match="tokens and parents"):
            beam_finish(st._replace(step=4), a, b, **args)
    with pytest.raises(ValueError, match="num_beams"):
        expand_states([x], 0)
    with pytest.raises(ValueError, match="groups"):
        reorder_states_([x], torch.arange(6), 4)


def test_no_cpu_path():
    st = beam_start(2, 3, "cpu")
    args = dict(eos_token_id=1, pad_token_id=0)
    t, p = torch.zeros(0, 6, dtype=torch.int64), torch.zeros(0, 6, dtype=torch.int32)
    for call in (lambda: beam_step(torch.zeros(6, 50), st, **args),
                 lambda: beam_finish(st, t, p, **args),
                 lambda: reorder_states_([torch.zeros(6, 2)], torch.arange(6), 3),
                 lambda: expand_states([torch.zeros(6, 2)], 3),
                 lambda: dl.BeamDecodeState(torch.zeros(2, 4, dtype=torch.int64), 3, 1, 0, 5, 1.0,
                                            False)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_counts_whose_rows_would_wrap():
    """groups * beams past 64 bits, to few or to none."""
    L = lib()
    for groups in ((1 << 62), (1 << 62) + 2, (1 << 61) + (1 << 20)):
        r = rows(groups=groups, done=4096)
        assert L.gtp_beam_workspace_bytes(r) == 0
        assert L.gtp_beam_candidates(r, 4096, 4096, 4096, None, 4096, 1 << 40, None) == UNSUPPORTED
        assert L.gtp_beam_step(r, state(), None, 4096, 1 << 40, None) == UNSUPPORTED
        assert L.gtp_beam_advance(4096, 4096, 4096, groups, 4, 8, state(), None) == UNSUPPORTED
        assert L.gtp_beam_finish(*(4096,) * 7, groups, 4, 5, 1.0, 1, 0, 2, *(4096,) * 3, 5,
                                 None) == UNSUPPORTED
        shape = Shape(64, 64, (I64 * 4)(1, 1, 1, 1), (I64 * 4)(0, 0, 0, 0))
        p = (VP * 1)(4096)
        assert L.gtp_reorder_states(p, 1, shape, 4096, groups, 4, None, None) == UNSUPPORTED
        assert L.gtp_expand_states(p, p, 1, shape, groups, 4, None) == UNSUPPORTED
