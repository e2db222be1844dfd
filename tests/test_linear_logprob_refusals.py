"""Calls that the hidden-state losses refuse, without a GPU."""

import ctypes

import pytest
import torch

import graspo_amd
from graspo_amd.graspo_loss import sequence_log_probs_from_hidden
from graspo_amd.sft_loss import sft_cross_entropy_loss_from_hidden

BF = torch.bfloat16
VP, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32


def test_shapes_and_types_are_refused():
    h, w = torch.zeros(2, 5, 16, dtype=BF), torch.zeros(9, 16, dtype=BF)
    t = torch.zeros(2, 5, dtype=torch.int64)
    for hid, wt in ((h.float(), w.float()), (h, w.half()), (h.half(), w), (h.double(), w.double())):
        with pytest.raises(ValueError, match="bfloat16"):
            sequence_log_probs_from_hidden(hid, wt, t)
        with pytest.raises(ValueError, match="bfloat16"):
            sft_cross_entropy_loss_from_hidden(hid, wt, t)
    with pytest.raises(ValueError, match="weight"):
        sequence_log_probs_from_hidden(h, torch.zeros(9, 15, dtype=BF), t)
    with pytest.raises(ValueError, match="weight"):
        sequence_log_probs_from_hidden(h, torch.zeros(9, 16, 1, dtype=BF), t)
    with pytest.raises(ValueError, match="output ids"):
        sequence_log_probs_from_hidden(h, w, t[:, :4])
    with pytest.raises(ValueError, match="labels"):
        sft_cross_entropy_loss_from_hidden(h, w, t[:, :4])
    with pytest.raises(ValueError, match="labels"):
        sft_cross_entropy_loss_from_hidden(h[0], w, t[0])


def test_no_cpu_path():
    h, w = torch.zeros(2, 5, 16, dtype=BF), torch.zeros(9, 16, dtype=BF)
    t = torch.zeros(2, 5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sequence_log_probs_from_hidden(h, w, t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sft_cross_entropy_loss_from_hidden(h, w, t)


class LinearRows(ctypes.Structure):
    _fields_ = [("hidden", VP), ("weight", VP), ("targets", VP), ("dtype", I32),
                ("targets_int64", I32), ("has_ignore", I32), ("ignore_index", I64), ("B", I64),
                ("S", I64), ("T", I64), ("K", I64), ("V", I64), ("hidden_batch_stride", I64),
                ("hidden_row_stride", I64), ("weight_stride", I64), ("target_batch_stride", I64),
                ("target_row_stride", I64)]


GOOD = dict(hidden=4096, weight=4096, targets=4096, dtype=1, targets_int64=1, B=2, S=8, T=8, K=64,
            V=100, hidden_batch_stride=512, hidden_row_stride=64, weight_stride=64,
            target_batch_stride=8, target_row_stride=1)
INVALID, UNSUPPORTED = 1, 2


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), INVALID), (dict(T=9), INVALID), (dict(K=0), INVALID), (dict(V=0), INVALID),
    (dict(weight_stride=32), INVALID), (dict(hidden_row_stride=-64), INVALID),
    (dict(target_row_stride=-1), INVALID), (dict(hidden=0), INVALID), (dict(weight=0), INVALID),
    (dict(targets=0), INVALID), (dict(dtype=0), UNSUPPORTED), (dict(dtype=9), UNSUPPORTED),
    (dict(weight=4104), UNSUPPORTED), (dict(weight_stride=65), UNSUPPORTED),
    (dict(weight_stride=1 << 22), UNSUPPORTED), (dict(K=60, weight_stride=60), UNSUPPORTED),
    (dict(B=2048, S=2048, T=2048), UNSUPPORTED), (dict(V=1 << 31), UNSUPPORTED),
    (dict(K=1 << 22, weight_stride=1 << 22), UNSUPPORTED),
    (dict(V=2000000000, S=200000, T=200000), UNSUPPORTED),
])
def test_c_entry_points_refuse(change, code):
    """Each of these returns its code before anything is launched."""
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    for f in (L.gtp_linear_logprob_workspace_bytes, L.gtp_linear_logprob_backward_workspace_bytes):
        f.restype, f.argtypes = ctypes.c_size_t, [ctypes.POINTER(LinearRows)]
    L.gtp_linear_logprob_rows.argtypes = [ctypes.POINTER(LinearRows), VP, VP, VP, VP, VP, VP,
                                          ctypes.c_size_t, VP]
    L.gtp_linear_logprob_backward.argtypes = [ctypes.POINTER(LinearRows), VP, VP, VP, VP, VP, VP,
                                              ctypes.c_size_t, VP]
    r = LinearRows(**{**GOOD, **change})
    assert L.gtp_linear_logprob_workspace_bytes(ctypes.byref(r)) == 0
    assert L.gtp_linear_logprob_backward_workspace_bytes(ctypes.byref(r)) == 0
    big = 1 << 40
    assert L.gtp_linear_logprob_rows(ctypes.byref(r), 4096, 4096, None, None, None, 4096, big,
                                     None) == code
    assert L.gtp_linear_logprob_backward(ctypes.byref(r), 4096, 4096, None, 4096, 4096, 4096, big,
                                         None) == code


def test_c_entry_points_refuse_buffers():
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    L.gtp_linear_logprob_workspace_bytes.restype = ctypes.c_size_t
    r = LinearRows(**GOOD)
    need = L.gtp_linear_logprob_workspace_bytes(ctypes.byref(r))
    assert need > 0
    f = L.gtp_linear_logprob_rows
    f.argtypes = [ctypes.POINTER(LinearRows), VP, VP, VP, VP, VP, VP, ctypes.c_size_t, VP]
    p = ctypes.byref(r)
    assert f(p, None, 4096, None, None, None, 4096, need, None) == INVALID
    assert f(p, 4096, None, None, None, None, 4096, need, None) == INVALID
    assert f(p, 4096, 4096, 4096, None, None, 4096, need, None) == INVALID
    assert f(p, 4096, 4096, None, None, None, None, need, None) == INVALID
    assert f(p, 4096, 4096, None, None, None, 4096, need - 1, None) == INVALID
