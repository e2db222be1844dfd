"""The embedding lookup and its table's gradient against the formulas in 64
bits.

Tolerances, from u = finfo(type).eps / 2 (0 for fp32, whose rounding is w)
and w = 2^-24: a row is one fp32 product rounded once, (w + u) |row|; a
gradient row sums its c tokens in fp32, c w sum|g|, times the scale, and is
rounded once, (2 w + u) of its size and half the type's smallest step.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.embedding import token_embedding

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
IDS = ["bf16", "fp16", "fp32"]


def half_step(dtype):
    return 0.0 if dtype == FP else torch.finfo(dtype).eps / 2


def expect(ids, grad, V, scale, padding=None, base=None):
    """(gradient, bound) in 64 bits; grad [N, H] CPU."""
    H = grad.shape[1]
    live = torch.ones_like(ids, dtype=torch.bool) if padding is None else ids != padding
    i, g = ids[live].long(), grad[live].double()
    want = torch.zeros(V, H, dtype=torch.float64).index_add_(0, i, g) * scale
    mag = torch.zeros(V, H, dtype=torch.float64).index_add_(0, i, g.abs()) * abs(scale)
    count = torch.bincount(i, minlength=V).double()[:, None]
    if base is not None:
        want, mag = want + base.double(), mag + base.double().abs()
    tiny = torch.finfo(grad.dtype).smallest_normal * torch.finfo(grad.dtype).eps / 2
    err = count * W * mag
    return want, err + (2 * W + half_step(grad.dtype)) * (want.abs() + err) + tiny * (count > 0)


def check(got, want, err):
    bad = ~((got.cpu().double() - want).abs() <= err)
    assert not bool(bad.any()), int(bad.sum())


def ids_of(N, V, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "zipf":
        return ((V + 1.0) ** torch.rand(N, generator=g, dtype=torch.float64) - 1).long().clamp(0, V - 1)
    if kind == "same":
        return torch.full((N,), V - 1)
    if kind == "each once":
        return torch.randperm(V, generator=g)[:N]
    return torch.randint(0, V, (N,), generator=g)


SIZES = [
    # N, V, H
    (1, 1, 1), (1, 50, 8), (2, 3, 16), (7, 600, 33), (64, 513, 256), (65, 1000, 1027),
    (300, 511, 72), (1000, 512, 136), (999, 262143, 24), (1025, 262144, 8), (4097, 70000, 40),
    (20000, 9, 64), (33000, 151936, 16), (130, 40, 4104),
]


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=IDS)
@pytest.mark.parametrize("N,V,H", SIZES)
def test_rows_and_gradient(N, V, H, dtype):
    g = torch.Generator().manual_seed(N + V)
    w = torch.randn(V, H, generator=g).to(dtype)
    grad = torch.randn(N, H, generator=g).to(dtype)
    ids = ids_of(N, V, N)
    scale = 1.0 if N % 2 else 11.3137
    wd = w.cuda().requires_grad_()
    out = token_embedding(ids.cuda(), wd, scale=scale)
    assert out.dtype == dtype and out.shape == (N, H)
    s32 = float(torch.tensor(scale, dtype=FP))
    want = w[ids].double() * s32
    u = half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    check(out.detach(), want, (W + u) * want.abs() + tiny)
    if scale == 1.0:
        assert torch.equal(out.detach().cpu(), w[ids])
    (gw,) = torch.autograd.grad(out, [wd], grad.cuda())
    assert gw.dtype == dtype
    check(gw, *expect(ids, grad, V, s32))


@pytest.mark.parametrize("kind", ["same", "each once", "uniform"])
@pytest.mark.parametrize("N", [31, 32, 33, 1000])
def test_runs_of_ids(N, kind):
    """One run over every chunk, runs of one, and chance."""
    V, H = 1200, 48
    ids = ids_of(N, V, 3, kind)
    grad = torch.randn(N, H, generator=torch.Generator().manual_seed(N))
    got = ops.embedding_backward(ids.cuda(), grad.cuda(), V)
    check(got, *expect(ids, grad, V, 1.0))


def test_runs_that_cross_one_border_each():
    """Runs of every length from 1 to 70, so that borders fall everywhere."""
    ids = torch.cat([torch.full((n,), n) for n in range(1, 71)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1))]
    grad = torch.randn(ids.numel(), 40, generator=torch.Generator().manual_seed(2))
    for es in (BF, FP):
        got = ops.embedding_backward(ids.cuda(), grad.to(es).cuda(), 72)
        check(got, *expect(ids, grad.to(es), 72, 1.0))


@pytest.mark.parametrize("padding", [0, 5, -1])
def test_padding_has_no_gradient(padding):
    B, S, V, H = 3, 50, 80, 64
    ids = ids_of(B * S, V, 4).view(B, S)
    ids[1, 20:] = padding % V
    w = torch.randn(V, H).to(BF)
    grad = torch.randn(B, S, H).to(BF)
    wd = w.cuda().requires_grad_()
    out = token_embedding(ids.cuda(), wd, padding_idx=padding)
    assert out.shape == (B, S, H) and torch.equal(out.detach().cpu(), w[ids])
    (gw,) = torch.autograd.grad(out, [wd], grad.cuda())
    assert bool((gw[padding % V] == 0).all())
    check(gw, *expect(ids.reshape(-1), grad.view(-1, H), V, 1.0, padding % V))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_added_to_a_tied_gradient(dtype):
    """`out` keeps the rows without a token to the bit, whatever they hold."""
    N, V, H = 500, 900, 56
    ids = ids_of(N, V, 6)
    g = torch.Generator().manual_seed(6)
    grad, base = torch.randn(N, H, generator=g).to(dtype), torch.randn(V, H, generator=g).to(dtype)
    used = torch.zeros(V, dtype=torch.bool).index_fill_(0, ids, True)
    base[~used] = float("nan")
    to = base.cuda()
    got = ops.embedding_backward(ids.cuda(), grad.cuda(), V, scale=2.0, out=to)
    assert got.data_ptr() == to.data_ptr()
    assert bool(to.cpu()[~used].isnan().all())
    want, err = expect(ids, grad, V, 2.0, base=torch.where(used[:, None], base, torch.zeros(())))
    check(to.cpu()[used], want[used], err[used])
    # views behind an odd element are added to as well
    odd = torch.zeros(1 + V * H, dtype=dtype, device="cuda")[1:].view(V, H)
    ops.embedding_backward(ids.cuda(), grad.cuda(), V, out=odd)
    check(odd, *expect(ids, grad, V, 1.0))


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=IDS)
@pytest.mark.parametrize("N,V,H", SIZES)
def test_the_order_stands_for_the_ids(N, V, H, dtype):
    """To the bit, twice from one order, into new memory and onto old."""
    ids = ids_of(N, V, N + H).cuda()
    if N > 3:
        ids[1], ids[-1] = -1, V
    w, grad = torch.randn(V, H).to(dtype).cuda(), torch.randn(N, H).to(dtype).cuda()
    out, bad, order = ops.embedding_ordered(ids, w, scale=3.0, padding_idx=V // 2, check=False)
    assert not bad and order.dtype == torch.int32
    assert torch.equal(out.nan_to_num(7.0), ops.embedding(ids, w, scale=3.0, check=False)[0].nan_to_num(7.0))
    want = ops.embedding_backward(ids, grad, V, scale=3.0, padding_idx=V // 2)
    ids.zero_()
    for _ in range(2):
        assert torch.equal(ops.embedding_backward(None, grad, V, scale=3.0, order=order), want)
    onto = torch.zeros(V, H, dtype=dtype, device="cuda")
    ops.embedding_backward(None, grad, V, scale=3.0, order=order, out=onto)
    assert torch.equal(onto, want)


def test_rows_without_tokens_are_zeros():
    """Whatever the memory held, at every alignment of a row; nothing behind
    the last row is written."""
    for H in (1, 3, 7, 9, 64, 129, 1027):
        for dtype in (BF, FP):
            V, N = 203, 3
            ids = torch.tensor([0, V - 1, 77], device="cuda")
            w = torch.zeros(V, H, dtype=dtype, device="cuda")
            grad = torch.ones(N, H, dtype=dtype, device="cuda")
            order = ops.embedding_ordered(ids, w)[2]
            dirty = torch.full((V * H + 1024,), float("nan"), dtype=dtype, device="cuda")
            del dirty  # the allocator hands this block out next
            for got in (ops.embedding_backward(ids, grad, V),
                        ops.embedding_backward(None, grad, V, order=order)):
                want = torch.zeros(V, H)
                want[ids.cpu()] = 1.0
                assert torch.equal(got.cpu().float(), want)


def test_orders_of_other_sizes_are_refused():
    w = torch.zeros(40, 8, device="cuda")
    order = ops.embedding_ordered(torch.arange(5, device="cuda"), w)[2]
    grad = torch.zeros(5, 8, device="cuda")
    for g, V, o in ((grad[:4], 40, order), (grad, 99, order), (grad, 40, order.long()),
                    (grad, 40, order[:-1]), (grad, 40, order.cpu())):
        with pytest.raises(RuntimeError, match="order"):
            ops.embedding_backward(None, g, V, order=o)
    with pytest.raises(RuntimeError, match="neither"):
        ops.embedding_backward(None, grad, 40)


def test_layouts():
    N, V, H = 90, 200, 64
    ids = ids_of(N, V, 7)
    w = torch.randn(V, H).to(BF)
    grad = torch.randn(N, H).to(BF)
    want = ops.embedding(ids.cuda(), w.cuda())[0]
    gwant = ops.embedding_backward(ids.cuda(), grad.cuda(), V)
    wide = torch.nn.functional.pad(w, (0, 3)).cuda()[:, :H]
    for x in (w.cuda().t().contiguous().t(), wide, torch.cat([w, w], 1).cuda()[:, :H]):
        assert not x.is_contiguous()
        assert torch.equal(ops.embedding(ids.cuda(), x)[0], want)
    strided = torch.stack([ids, ids], 1).cuda()[:, 0]
    for i in (ids.int().cuda(), strided, ids.cuda().view(9, 10).t().contiguous().t()):
        assert torch.equal(ops.embedding(i, w.cuda())[0].view(N, H), want)
        assert torch.equal(ops.embedding_backward(i, grad.cuda().view(*i.shape, H), V), gwant)
    gpad = torch.nn.functional.pad(grad, (0, 5)).cuda()[:, :H]
    for g in (grad.cuda().t().contiguous().t(), gpad):
        assert torch.equal(ops.embedding_backward(ids.cuda(), g, V), gwant)
    # a sum's gradient is one row for all
    wd = w.cuda().requires_grad_()
    (gw,) = torch.autograd.grad(token_embedding(ids.cuda(), wd).sum(), [wd])
    count = torch.bincount(ids, minlength=V).float()
    assert torch.equal(gw.cpu().float(), count[:, None].expand(V, H).to(BF).float())


def test_the_same_bits_every_time():
    ids, grad = ids_of(5000, 300, 8).cuda(), torch.randn(5000, 128, device="cuda")
    first = ops.embedding_backward(ids, grad, 300)
    for _ in range(5):
        assert torch.equal(ops.embedding_backward(ids, grad, 300), first)


def test_nothing_to_look_up():
    w = torch.randn(10, 8, device="cuda", requires_grad=True)
    ids = torch.empty(2, 0, dtype=torch.int64, device="cuda")
    out = token_embedding(ids, w)
    assert out.shape == (2, 0, 8)
    (gw,) = torch.autograd.grad(out.sum(), [w])
    assert bool((gw == 0).all())
    scalar = token_embedding(torch.tensor(3, device="cuda"), w)
    assert torch.equal(scalar, w[3].detach())


@pytest.mark.parametrize("bad", [-1, 50, 2 ** 31 + 3])
def test_bad_ids(bad):
    w = torch.randn(50, 16, device="cuda").to(BF).requires_grad_()
    ids = torch.arange(20, device="cuda")
    ids[4] = bad
    with pytest.raises(RuntimeError, match="outside"):
        token_embedding(ids, w)
    out = token_embedding(ids, w, check_status=False)
    rest = torch.arange(20, device="cuda") != 4
    assert bool(out[4].isnan().all()) and torch.equal(out[rest].detach(), w[ids[rest]].detach())
    (gw,) = torch.autograd.grad(out, [w], torch.ones_like(out))
    assert bool((gw[:20][rest] == 1).all()) and bool((gw[4] == 0).all()) and bool((gw[20:] == 0).all())


def test_a_table_past_32_bit_offsets():
    V, H = (1 << 31) // 1024 + 1000, 1024
    ids = torch.tensor([V - 1, 0, V - 2, (1 << 31) // 1024, V - 1], device="cuda")
    w = torch.zeros(V, H, dtype=BF, device="cuda")
    w[ids] = torch.arange(1.0, 6.0, device="cuda", dtype=BF)[:, None]
    w[V - 1] = 7.0
    w.requires_grad_()
    out = token_embedding(ids, w)
    assert out.detach()[:, 5].tolist() == [7.0, 2.0, 3.0, 4.0, 7.0]
    (gw,) = torch.autograd.grad(out, [w], torch.ones_like(out))
    assert gw[ids].float().mean(1).tolist() == [2.0, 1.0, 1.0, 1.0, 2.0]
    gw[ids] = 0
    assert not bool(gw.any())


def test_one_order_on_two_streams():
    ids, w = ids_of(3000, 500, 21).cuda(), torch.randn(500, 96, device="cuda")
    grads = [torch.randn(3000, 96, device="cuda") for _ in range(2)]
    order = ops.embedding_ordered(ids, w)[2]
    want = [ops.embedding_backward(ids, g, 500) for g in grads]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, g in zip(streams, grads):
            with torch.cuda.stream(s):
                got.append(ops.embedding_backward(None, g, 500, order=order))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])


def test_captured_and_replayed():
    N, V, H = 300, 700, 64
    ids = torch.zeros(N, dtype=torch.int64, device="cuda")
    w, grad = torch.zeros(V, H, device="cuda"), torch.zeros(N, H, device="cuda")

    def fill(k):
        ids.copy_(ids_of(N, V, 50 + k))
        w.normal_(), grad.normal_()

    def step():
        out, _, order = ops.embedding_ordered(ids, w, scale=3.0)
        return (ops.embedding(ids, w, scale=3.0)[0], out,
                ops.embedding_backward(ids, grad, V, scale=3.0),
                ops.embedding_backward(None, grad, V, scale=3.0, order=order))

    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        fill(k)
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    """fp64 differences of sum(g * rows) over the table's fp32 values."""
    ids = torch.tensor([3, 1, 3, 0, 3])
    g = torch.randn(5, 6, dtype=torch.float64)
    w = torch.randn(4, 6, dtype=torch.float64)
    f = lambda t: (g * t[ids] * 2.5).sum()  # noqa: E731
    got = ops.embedding_backward(ids.cuda(), g.float().cuda(), 4, scale=2.5).cpu().double()
    for v in range(4):
        for c in range(6):
            d = torch.zeros_like(w)
            d[v, c] = 1e-4
            assert abs(float((f(w + d) - f(w - d)) / 2e-4) - float(got[v, c])) < 1e-5
