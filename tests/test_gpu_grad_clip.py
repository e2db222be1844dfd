"""The global gradient norm and clipping against the formulas in 64 bits.

Tolerances: the norm's sums are 64-bit and it is rounded once to fp32, w =
2^-24 (and n 2^-53, below 1e-9 here).  The factor is three fp32 operations on
that norm (its addition, the division, the norm's own rounding), a clipped
element one more and one rounding to its type: 5 w + u with u =
finfo(type).eps / 2 (0 for fp32), and half the type's smallest step.
"""

from __future__ import annotations

import math

import pytest
import torch

from graspo_amd import ops
from graspo_amd.grad_clip import clip_grad_norm_, clip_grads_with_norm_, get_total_norm

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def exact_norm(tensors, p):
    xs = [t.detach().cpu().double().reshape(-1) for t in tensors]
    x = torch.cat(xs) if xs else torch.zeros(0, dtype=torch.float64)
    if x.numel() == 0:
        return 0.0
    if p == math.inf:
        return float(x.abs().max())
    return float(x.abs().sum() if p == 1 else x.square().sum().sqrt())


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        out.append(p)
    return out


def check_clipped(got, before, norm, max_norm):
    f = min(1.0, max_norm / (norm + 1e-6))
    for a, b in zip(got, before):
        want = b.double() * f
        if f == 1.0:
            assert torch.equal(a.cpu(), b)
            continue
        u = 0.0 if b.dtype == FP else torch.finfo(b.dtype).eps / 2
        tiny = torch.finfo(b.dtype).smallest_normal * torch.finfo(b.dtype).eps / 2
        assert bool(((a.cpu().double() - want).abs() <= (5 * W + u) * want.abs() + tiny).all())


def some(shapes, dtypes, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * spread).to(d) for s, d in zip(shapes, dtypes)]


LISTS = {
    "one element": ([(1,)], [FP]),
    "scalar": ([()], [BF]),
    "mixed": ([(3, 5), (70000,), (1,), (257, 129), (16,)], [FP, BF, HF, BF, FP]),
    "empty among them": ([(0,), (33,), (4, 0), (7, 9)], [FP, BF, HF, FP]),
    "many": ([(i % 37 + 1, 11) for i in range(500)], [(FP, BF, HF)[i % 3] for i in range(500)]),
    "chunk borders": ([(16384,), (16385,), (16383,), (32768,), (4,), (65536 + 3,)], [FP] * 6),
    "half chunk borders": ([(32768,), (32769,), (32767,), (65536,), (8,), (131072 + 7,)], [BF] * 6),
    "kernel argument borders": ([(9,)] * 193, [FP] * 193),
    "large": ([(3000, 1111), (1 << 22,)], [FP, BF]),
}


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("which", list(LISTS))
def test_norm_and_clip(which, p):
    before = some(*LISTS[which], seed=len(which))
    grads = [t.cuda() for t in before]
    norm = exact_norm(before, p)
    for max_norm in (norm * 0.37 + 1e-3, norm * 2 + 1.0):
        work = [t.clone() for t in grads]
        got = clip_grad_norm_(params_of(work), max_norm, norm_type=p)
        assert got.dtype == FP and got.dim() == 0
        assert abs(float(got) - norm) <= (W + 1e-9) * norm
        check_clipped(work, before, norm, max_norm)
    assert torch.equal(get_total_norm(grads, p), got)
    work = [t.clone() for t in grads]
    clip_grads_with_norm_(params_of(work), 0.25 * norm, got)
    check_clipped(work, before, norm, 0.25 * norm)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("off", range(0, 9))
def test_views_at_every_alignment(dtype, off):
    """Views of one bucket, whose neighbours stay as they are."""
    sizes = [1, 2, 7, 8, 9, 4096 * 8, 5, 65536 + 9, 3]
    flat = torch.randn(off + sum(sizes) + 5, generator=torch.Generator().manual_seed(off)).to(dtype)
    for n in (16400, 2):  # and tensors that end behind a whole chunk and a boundary
        sizes[5] = n * 8
        total = off + sum(sizes) + 5
        flat = torch.randn(total, generator=torch.Generator().manual_seed(off)).to(dtype)
        dev = flat.cuda()
        views, at = [], off
        for k in sizes:
            views.append(dev[at : at + k])
            at += k
        before = [v.cpu().clone() for v in views]
        norm = exact_norm(before, 2)
        got = clip_grad_norm_(params_of(views), 0.5 * norm)
        assert abs(float(got) - norm) <= (W + 1e-9) * norm
        check_clipped(views, before, norm, 0.5 * norm)
        assert torch.equal(dev[:off].cpu(), flat[:off]) and torch.equal(dev[at:].cpu(), flat[at:])


@pytest.mark.parametrize("dtype,per", [(FP, 4), (BF, 8)])
@pytest.mark.parametrize("extra", [-1, 0, 1, 2, 3, 5, 7, 9])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_every_element_counts_once(dtype, per, extra, off):
    """Ones around whole chunks of 4096 vectors: the norm's square is their
    number."""
    n = 4096 * per + extra
    flat = torch.zeros(off + n + 8, dtype=dtype, device="cuda")
    flat[off : off + n] = 1.0
    got = ops.grad_norm([flat[off : off + n]], 1.0)
    assert float(got) == n


def test_values_beyond_fp32_squares():
    big = torch.full((1000,), 3e38, device="cuda")
    assert float(get_total_norm([big[:1]])) == pytest.approx(3e38, rel=1e-6)
    small = torch.full((10000,), 1e-30, device="cuda")
    assert float(get_total_norm([small])) == pytest.approx(1e-28, rel=1e-6)
    p = params_of([big])
    # the norm itself passes fp32's range: infinite, and everything becomes 0
    assert float(clip_grad_norm_(p, 1.0)) == math.inf
    assert bool((p[0].grad == 0).all())


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_nan_and_infinity(p):
    for v in (float("nan"), math.inf, -math.inf):
        x = torch.randn(70000)
        x[69999] = v
        g = [torch.randn(10, device="cuda"), x.cuda()]
        with pytest.raises(RuntimeError, match="non-finite"):
            clip_grad_norm_(params_of(g), 1.0, norm_type=p, error_if_nonfinite=True)
        assert torch.equal(g[1].cpu().nan_to_num(9.0), x.nan_to_num(9.0))  # untouched
        with pytest.raises(RuntimeError, match="non-finite"):
            get_total_norm(g, p, error_if_nonfinite=True)
        norm = clip_grad_norm_(params_of(g), 1.0, norm_type=p)
        if v != v:
            assert bool(norm.isnan()) and bool(g[0].isnan().all()) and bool(g[1].isnan().all())
        else:  # inf * 0
            assert float(norm) == math.inf and bool((g[0] == 0).all())
            assert bool(g[1][69999].isnan()) and bool((g[1][:69999] == 0).all())


def test_layouts():
    base = torch.randn(60, 80, generator=torch.Generator().manual_seed(1))
    dense = base.cuda().t()                       # no gaps, other order
    gaps = torch.zeros(60, 100, device="cuda")
    gaps[:, 80:] = 7.0
    gaps[:, :80] = base.cuda()
    view = gaps[:, :80]
    norm = exact_norm([base, base], 2)
    got = clip_grad_norm_([_holder(dense), _holder(view)], 0.5 * norm)
    assert abs(float(got) - norm) <= (W + 1e-9) * norm
    check_clipped([dense.t(), view], [base, base], norm, 0.5 * norm)
    assert bool((gaps[:, 80:] == 7.0).all())


class _holder:
    """What the functions need of a parameter: its gradient."""

    def __init__(self, grad):
        self.grad = grad


def test_max_norm_of_zero_and_no_gradient():
    g = torch.randn(100, device="cuda")
    clip_grad_norm_(_as_param(g), 0.0)
    assert bool((g == 0).all())
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(get_total_norm([])) == 0.0
    assert float(get_total_norm([torch.empty(0, device="cuda")])) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_of_a_bucket(dtype):
    """Neighbours in any order, empty ones and gaps between: each element of
    the listed views counts and is scaled once, the others stay."""
    sizes = [5, 0, 4096, 1, 70001, 33, 16384, 9, 2, 65536]
    bucket = torch.randn(sum(sizes) + 7, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    before, at, views = bucket.clone(), 3, []
    for n in sizes:
        views.append(bucket[at : at + n])
        at += n
    for order in (range(10), [9, 8, 7, 6, 5, 4, 3, 2, 1, 0], [0, 1, 2, 4, 5, 3, 7, 8], [6, 7, 9]):
        listed = [views[i] for i in order]
        bucket.copy_(before)
        want = exact_norm([v.clone() for v in listed], 2.0)
        norm = clip_grad_norm_([_as_param(v) for v in listed], 1.0)
        assert abs(float(norm) - float(want)) <= 2 * 2.0 ** -24 * float(want)
        # the same products one tensor at a time
        alone = before.clone()
        for v in listed:
            w = alone[v.storage_offset() : v.storage_offset() + v.numel()]
            clip_grads_with_norm_([_as_param(w)], 1.0, norm)
        assert torch.equal(bucket, alone)


def test_a_tensor_past_32_bit_offsets():
    n = (1 << 31) + 4099
    x = torch.ones(n, dtype=BF, device="cuda")
    norm = clip_grad_norm_([_as_param(x)], 0.25 * math.sqrt(n))
    assert abs(float(norm) - math.sqrt(n)) <= 2 * W * math.sqrt(n)
    assert bool((x == 0.25).all())


def _as_param(g):
    p = torch.nn.Parameter(torch.zeros_like(g))
    p.grad = g
    return p


def test_overlaps_are_refused():
    x = torch.randn(100, device="cuda")
    keep = x.clone()
    for grads in ([x, x], [x[:60], x[50:]], [x[50:], x[:60]], [x[:1].expand(5)]):
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grad_norm_([_holder(g) for g in grads], 1e-3)
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads_with_norm_([_holder(g) for g in grads], 1e-3, torch.tensor(1.0, device="cuda"))
    assert torch.equal(x, keep)
    # the norm alone may read what it likes
    assert float(get_total_norm([x, x])) == pytest.approx(math.sqrt(2) * float(keep.norm()), rel=1e-5)
    # neighbours do not overlap
    clip_grad_norm_([_holder(x[50:]), _holder(x[:50])], 1e-3)


def test_refused_types():
    for t in (torch.zeros(3, dtype=torch.float64, device="cuda"),
              torch.zeros(3, dtype=torch.int32, device="cuda")):
        with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
            get_total_norm([t])
    with pytest.raises(RuntimeError, match="every tensor|GPU"):
        get_total_norm([torch.zeros(3, device="cuda"), torch.zeros(3)])


def test_sparse_gradients_are_refused():
    dense = torch.ones(4, 4, device="cuda")
    for tensors in ([dense.to_sparse()], [dense, dense.to_sparse()]):
        with pytest.raises(ValueError, match="sparse"):
            get_total_norm(tensors)


def test_captured_and_replayed():
    shapes = [(300, 70), (5,), (33, 33)] * 70
    grads = [torch.zeros(s, device="cuda") for s in shapes]
    ps = params_of(grads)

    def fill(k):
        g = torch.Generator(device="cuda").manual_seed(k)
        for t in grads:
            t.normal_(generator=g).mul_(0.1 ** k)

    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        clip_grad_norm_(ps, 1.0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = clip_grad_norm_(ps, 1.0)
    for k in range(5):
        fill(k)
        want_norm = clip_grad_norm_(ps, 1.0)
        want = [t.clone() for t in grads]
        fill(k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want_norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
