"""Calls that the low-rank adapters refuse, without a GPU."""

import ctypes

import pytest
import torch

import graspo_amd
from graspo_amd.lora import lora_add

VP, I64, I32, SZ, F32 = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t,
                         ctypes.c_float)
OK, INVALID, UNSUPPORTED = 0, 1, 2


class Lora(ctypes.Structure):
    _fields_ = [(n, VP) for n in ("x", "base", "y", "a", "b", "scales", "ids")] + [
        (n, I64) for n in ("requests", "rows", "k", "n", "x_stride", "base_stride")] + [
        (n, I32) for n in ("dtype", "ids_int64", "rank", "adapters")] + [("scale", F32)]


class Grads(ctypes.Structure):
    _fields_ = [("grad", VP), ("grad_stride", I64), ("grad_x", VP), ("grad_a", VP), ("grad_b", VP)]


def lib():
    L = ctypes.CDLL(graspo_amd.LIB_PATH)
    P = ctypes.POINTER
    for f in (L.gtp_lora_state_bytes, L.gtp_lora_backward_workspace_bytes):
        f.argtypes, f.restype = [P(Lora)], SZ
    L.gtp_lora_add.argtypes = [P(Lora), VP, SZ, VP]
    L.gtp_lora_backward.argtypes = [P(Lora), P(Grads), VP, SZ, VP, SZ, VP]
    return L


def lora(**change):
    a = dict(x=4096, base=4096, y=4096, a=4096, b=4096, scales=4096, ids=4096, requests=3, rows=5,
             k=64, n=96, x_stride=64, base_stride=96, dtype=1, ids_int64=1, rank=8, adapters=2,
             scale=1.0)
    a.update(change)
    return Lora(**a)


def grads(**change):
    a = dict(grad=4096, grad_stride=96, grad_x=4096, grad_a=4096, grad_b=4096)
    a.update(change)
    return Grads(**a)


@pytest.mark.parametrize("change,code", [
    (dict(requests=-1), INVALID), (dict(rows=-1), INVALID), (dict(k=0), INVALID),
    (dict(n=0), INVALID), (dict(rank=0), INVALID), (dict(adapters=0), INVALID),
    (dict(dtype=3), INVALID), (dict(ids=None), INVALID), (dict(rank=257), UNSUPPORTED),
    (dict(adapters=1025), UNSUPPORTED), (dict(k=(1 << 24) + 1), UNSUPPORTED),
    (dict(n=(1 << 24) + 1), UNSUPPORTED), (dict(requests=1 << 12, rows=1 << 12), UNSUPPORTED),
    (dict(adapters=1024, rank=256, k=1 << 24), UNSUPPORTED),
])
def test_sizes(change, code):
    L = lib()
    q = lora(**change)
    assert L.gtp_lora_state_bytes(q) == 0 and L.gtp_lora_backward_workspace_bytes(q) == 0
    assert L.gtp_lora_add(q, 4096, 1 << 40, None) == code
    assert L.gtp_lora_backward(q, grads(), 4096, 1 << 40, 4096, 1 << 40, None) == code


def test_pointers():
    L = lib()
    state, work = L.gtp_lora_state_bytes(lora()), L.gtp_lora_backward_workspace_bytes(lora())
    assert state > 0 and work > 0
    add = lambda q=None, s=4096, n=state: L.gtp_lora_add(lora() if q is None else q, s, n, None)  # noqa: E731
    back = lambda q=None, d=None, s=4096, n=state, w=4096, b=work: L.gtp_lora_backward(  # noqa: E731
        lora() if q is None else q, grads() if d is None else d, s, n, w, b, None)
    for name in ("x", "base", "y", "a", "b"):
        assert add(lora(**{name: None})) == add(lora(**{name: 4097})) == INVALID
        if name in ("x", "a", "b"):
            assert back(lora(**{name: None})) == back(lora(**{name: 4097})) == INVALID
    assert add(lora(x_stride=-1)) == add(lora(base_stride=-1)) == INVALID
    assert add(lora(scales=4098)) == add(lora(ids=4100)) == INVALID
    for s, n in ((None, state), (4104, state), (4096, state - 1)):
        assert add(s=s, n=n) == back(s=s, n=n) == INVALID
    for w, b in ((None, work), (4100, work), (4096, work - 1)):
        assert back(w=w, b=b) == INVALID
    for bad in (dict(grad=None), dict(grad=4097), dict(grad_stride=-1), dict(grad_x=4097),
                dict(grad_a=4097), dict(grad_b=4097)):
        assert back(d=grads(**bad)) == INVALID
    assert L.gtp_lora_backward(lora(), None, 4096, state, 4096, work, None) == INVALID
    assert L.gtp_lora_add(None, 4096, state, None) == INVALID
    empty = lora(requests=0, ids=None)
    assert L.gtp_lora_add(empty, None, 0, None) == OK
    assert L.gtp_lora_backward(empty, grads(), 4096, 256, 4096, 256, None) == UNSUPPORTED


def test_python_arguments():
    x, base = torch.zeros(3, 5, 8), torch.zeros(3, 5, 6)
    a, b = torch.zeros(2, 4, 8), torch.zeros(2, 6, 4)
    ids = torch.zeros(3, dtype=torch.int64)
    call = lambda base=base, x=x, a=a, b=b, ids=ids, **kw: lora_add(  # noqa: E731
        base, x, a, b, adapter_ids=ids, **kw)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        call(x=x.double())
    for bad in (dict(base=base.half()), dict(a=a.half()), dict(b=b.bfloat16())):
        with pytest.raises(ValueError, match="as x"):
            call(**bad)
    for bad in (dict(a=a[0]), dict(b=b[0]), dict(a=a[None]), dict(a=a[0, 0], b=b[0, 0])):
        with pytest.raises(ValueError, match="adapters"):
            call(**bad)
    for bad in (dict(x=x[..., :7]), dict(base=base[..., :5]), dict(base=base[:2]), dict(b=b[:1]),
                dict(a=a[:, :3]), dict(a=a[:0], b=b[:0]), dict(a=a[:, :0], b=b[..., :0])):
        with pytest.raises(ValueError, match="go together"):
            call(**bad)
    big = torch.zeros(1, 300, 8), torch.zeros(1, 6, 300)
    with pytest.raises(ValueError, match="rank 256"):
        call(a=big[0], b=big[1])
    with pytest.raises(ValueError, match="no adapter_ids"):
        call(ids=None)
    for bad in (ids.float(), ids.to(torch.int16)):
        with pytest.raises(ValueError, match="int32 or int64"):
            call(ids=bad)
    for bad in (ids[:2], ids[0], torch.zeros(3, 5, 8, dtype=torch.int64), ids.view(3, 1)):
        with pytest.raises(ValueError, match="leading"):
            call(ids=bad)
    for bad in (torch.ones(3), torch.ones(2, dtype=torch.float64), torch.ones(())):
        with pytest.raises(ValueError, match="scaling"):
            call(scaling=bad)
    with pytest.raises(ValueError, match="no gradient"):
        call(scaling=torch.ones(2, requires_grad=True))


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        lora_add(torch.zeros(3, 6), torch.zeros(3, 8), torch.zeros(4, 8), torch.zeros(6, 4))
