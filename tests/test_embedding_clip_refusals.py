"""Calls that the embedding and the gradient clipping refuse, without a GPU."""

import ctypes

import pytest
import torch

import graspo_amd
from graspo_amd import ops
from graspo_amd.embedding import token_embedding
from graspo_amd.grad_clip import clip_grad_norm_, clip_grads_with_norm_, get_total_norm

VP, I64, I32, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
INVALID, UNSUPPORTED = 1, 2


def test_embedding_arguments():
    ids, w = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(5, 4)
    for bad in (w[0], w[None]):
        with pytest.raises(ValueError, match="weight"):
            token_embedding(ids, bad)
    for dt in (torch.float64, torch.int32):
        with pytest.raises(ValueError, match="float32"):
            token_embedding(ids, w.to(dt))
    for dt in (torch.float32, torch.bool, torch.int16):
        with pytest.raises(ValueError, match="ids"):
            token_embedding(ids.to(dt), w)
    for pad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            token_embedding(ids, w, padding_idx=pad)
        with pytest.raises(ValueError, match="padding_idx"):
            ops.embedding_backward(ids, torch.zeros(2, 3, 4), 5, padding_idx=pad)


def test_clip_arguments():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    for kind in (0.0, 3.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_([p], 1.0, norm_type=kind)
        with pytest.raises(ValueError, match="norm_type"):
            get_total_norm([p.grad], kind)
    for most in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], most)
        with pytest.raises(ValueError, match="max_norm"):
            clip_grads_with_norm_([p], most, torch.tensor(1.0))
    sparse = torch.zeros(4, 4).to_sparse()
    with pytest.raises(ValueError, match="sparse"):
        get_total_norm([sparse])


def test_no_cpu_path():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    for call in (lambda: clip_grad_norm_([p], 1.0), lambda: get_total_norm([p.grad]),
                 lambda: clip_grads_with_norm_([p], 1.0, torch.tensor(1.0)),
                 lambda: token_embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(5, 4))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def _embedding_lib():
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    L.gtp_embedding_rows.argtypes = [VP, I32, I64, I64, VP, I32, I64, I64, I64, ctypes.c_float, VP, VP]
    L.gtp_embedding_backward.argtypes = [VP, I32, I64, I64, VP, I32, I64, I64, I64, ctypes.c_float,
                                         I64, I32, VP, VP, SZ, VP]
    L.gtp_embedding_backward_workspace_bytes.argtypes = [I32, I64, I64, I64]
    L.gtp_embedding_backward_workspace_bytes.restype = SZ
    return L


@pytest.mark.parametrize("change,code", [
    (dict(N=-1), INVALID), (dict(V=0), INVALID), (dict(H=0), INVALID), (dict(dtype=3), INVALID),
    (dict(ids=None), INVALID), (dict(stride=-1), INVALID), (dict(data=None), INVALID),
    (dict(out=None), INVALID), (dict(N=1 << 24), UNSUPPORTED), (dict(V=(1 << 31) - 1), UNSUPPORTED),
    (dict(H=1 << 25), UNSUPPORTED),
])
def test_embedding_entry_points(change, code):
    L = _embedding_lib()
    a = dict(ids=4096, N=8, stride=1, data=4096, dtype=1, V=100, H=64, out=4096)
    a.update(change)
    assert L.gtp_embedding_rows(a["ids"], 1, a["N"], a["stride"], a["data"], a["dtype"], a["V"],
                                a["H"], a["H"], 1.0, a["out"], None) == code
    assert L.gtp_embedding_backward(a["ids"], 1, a["N"], a["stride"], a["data"], a["dtype"], a["H"],
                                    a["V"], a["H"], 1.0, -1, 0, a["out"], 4096, 1 << 40, None) == code


def test_embedding_buffers():
    L = _embedding_lib()
    need = L.gtp_embedding_backward_workspace_bytes(1, 8, 100, 64)
    assert need > 0
    call = lambda out, ws, n, add=0: L.gtp_embedding_backward(  # noqa: E731
        4096, 1, 8, 1, 4096, 1, 64, 100, 64, 1.0, -1, add, out, ws, n, None)
    assert call(4096, 4096, need - 1) == INVALID
    assert call(4096, None, need) == INVALID
    assert call(4097, 4096, need) == INVALID      # no whole element
    assert call(4096, 4097, need) == INVALID
    assert L.gtp_embedding_rows(4096, 1, 8, 1, 4096, 1, 100, 64, 63, 1.0, 4096, None) == INVALID


def test_ordered_entry_points():
    L = _embedding_lib()
    L.gtp_embedding_order_bytes.argtypes = [I64, I64]
    L.gtp_embedding_order_bytes.restype = SZ
    L.gtp_embedding_backward_ordered_workspace_bytes.argtypes = [I32, I64, I64]
    L.gtp_embedding_backward_ordered_workspace_bytes.restype = SZ
    L.gtp_embedding_rows_ordered.argtypes = [VP, I32, I64, I64, VP, I32, I64, I64, I64,
                                             ctypes.c_float, VP, I64, VP, SZ, VP]
    L.gtp_embedding_backward_ordered.argtypes = [VP, SZ, I64, VP, I32, I64, I64, I64,
                                                 ctypes.c_float, I32, VP, VP, SZ, VP]
    need = L.gtp_embedding_order_bytes(8, 100)
    assert need == 4 * (4 * 8 + 4)  # two buffers of keys and places, and 100 bits
    assert L.gtp_embedding_order_bytes(0, 100) == L.gtp_embedding_order_bytes(8, 0) == 0
    rows = lambda order, n, N=8: L.gtp_embedding_rows_ordered(  # noqa: E731
        4096, 1, N, 1, 4096, 1, 100, 64, 64, 1.0, 4096, -1, order, n, None)
    ws = L.gtp_embedding_backward_ordered_workspace_bytes(1, 8, 64)
    grad = lambda order, n, N=8, w=4096, b=ws, out=4096: L.gtp_embedding_backward_ordered(  # noqa: E731
        order, n, N, 4096, 1, 64, 100, 64, 1.0, 0, out, w, b, None)
    for call in (rows, grad):
        assert call(None, need) == call(4097, need) == call(4096, need - 1) == INVALID
        assert call(4096, need, N=-1) == INVALID
        assert call(4096, 1 << 40, N=1 << 24) == UNSUPPORTED
    assert grad(4096, need, b=ws - 1) == grad(4096, need, w=None) == INVALID
    assert grad(4096, need, w=4098) == grad(4096, need, out=None) == INVALID


def test_norm_entry_points():
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    L.gtp_grad_norm_workspace_bytes.restype = SZ
    ptrs, sizes, types = (VP * 2)(4096, 8192), (I64 * 2)(10, 20), (ctypes.c_int32 * 2)(0, 1)
    L.gtp_grad_norm_workspace_bytes.argtypes = [VP, VP, VP, I64]
    L.gtp_grad_norm.argtypes = [VP, VP, VP, I64, I32, VP, VP, SZ, VP]
    L.gtp_clip_grads.argtypes = [VP, VP, VP, I64, VP, ctypes.c_float, VP]
    assert L.gtp_grad_norm_workspace_bytes(ptrs, sizes, types, 2) >= 16
    norm = lambda p, n, t, c, kind=2, out=4096, ws=4096, b=1 << 20: L.gtp_grad_norm(  # noqa: E731
        p, n, t, c, kind, out, ws, b, None)
    for bad in ((None, sizes, types, 2), (ptrs, None, types, 2), (ptrs, sizes, None, 2),
                (ptrs, sizes, types, -1),
                ((VP * 2)(4096, None), sizes, types, 2), ((VP * 2)(4097, 8192), sizes, types, 2),
                (ptrs, (I64 * 2)(10, -1), types, 2), (ptrs, sizes, (ctypes.c_int32 * 2)(0, 3), 2)):
        assert norm(*bad) == INVALID
        assert L.gtp_clip_grads(*bad, 4096, 1.0, None) == INVALID
        assert L.gtp_grad_norm_workspace_bytes(*bad) == 0
    assert norm(ptrs, (I64 * 2)(10, 1 << 40), types, 2) == UNSUPPORTED
    for kind in (0, 4):
        assert norm(ptrs, sizes, types, 2, kind=kind) == INVALID
    assert norm(ptrs, sizes, types, 2, out=None) == INVALID
    assert norm(ptrs, sizes, types, 2, ws=None) == INVALID
    assert norm(ptrs, sizes, types, 2, b=8) == INVALID
    assert L.gtp_clip_grads(ptrs, sizes, types, 2, None, 1.0, None) == INVALID
