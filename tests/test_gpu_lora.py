"""Low-rank adapters against the same in 64 bits, and their gradients.

u = 2^-24 (fp32), h = half a step of the dtype, g(n) = n u for a sum of n fp32
products in any order.  16-bit operands are exact in the products; a low-rank
value U is off by g(K) sum|x||a| and, as two parts, by 2^-16 |U| (hi and lo
carry 16 bits in bf16, 22 in fp16, as far as lo is a normal number: below that
2^-24 at most in fp16); the output by g(r) sum|U||b| more, and rounded once.
The gradients likewise, with V in U's place and sums over the rows.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.lora import lora_add

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(B, S, K, N, E, r, dtype, seed, none=0.2):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ids = torch.randint(0, E, (B,), generator=g)
    ids[torch.rand(B, generator=g) < none] = -1
    return dict(base=rnd(B, S, N).to(dtype), x=rnd(B, S, K).to(dtype),
                a=(rnd(E, r, K) / K ** 0.5).to(dtype), b=(rnd(E, N, r) * 0.5).to(dtype), ids=ids,
                s=torch.rand(E, generator=g) + 0.5, g=rnd(B, S, N).to(dtype))


def expect(d, dtype):
    """(value, bound) of the output and of x's, a's and b's gradients."""
    B, S, K = d["x"].shape
    E, r, _ = d["a"].shape
    N = d["b"].shape[1]
    dd = {k: v.double() for k, v in d.items() if k != "ids"}
    h = half_step(dtype)
    part = U if dtype == F4 else 2.0 ** -16
    tiny = 0.0 if dtype == F4 else torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    out, oe = dd["base"].clone(), torch.zeros(B, S, N, dtype=torch.float64)
    gx, gxe = torch.zeros(B, S, K).double(), torch.zeros(B, S, K).double()
    ga, gae = torch.zeros(E, r, K).double(), torch.zeros(E, r, K).double()
    gb, gbe = torch.zeros(E, N, r).double(), torch.zeros(E, N, r).double()
    for e in range(E):
        at = (d["ids"] == e).nonzero().flatten()
        if not len(at):
            continue
        n = len(at) * S
        s = float(d["s"][e])
        x, g = dd["x"][at].reshape(n, K), dd["g"][at].reshape(n, N)
        a, b = dd["a"][e], dd["b"][e]
        low = lambda y, w, size: (s * y @ w, (size + 8) * U * s * (y.abs() @ w.abs()))  # noqa: E731
        u, ue = low(x, a.t(), K)
        v, ve = low(g, b, N)
        ue, ve = ue + (part + 2 * U) * u.abs() + tiny, ve + (part + 2 * U) * v.abs() + tiny
        prod = lambda p, pe, w, k: (p @ w, (pe + (k + 8) * U * (p.abs() + pe)) @ w.abs())  # noqa: E731
        y, ye = prod(u, ue, b.t(), r)
        out[at] += y.view(len(at), S, N)
        oe[at] = (ye + U * (y.abs() + ye)).view(len(at), S, N)
        y, ye = prod(v, ve, a, r)
        gx[at], gxe[at] = y.view(len(at), S, K), ye.view(len(at), S, K)
        ga[e], t = prod(x.t(), torch.zeros(K, n), v, n)[0].t(), None
        gae[e] = (x.abs().t() @ (ve + (n + 8) * U * (v.abs() + ve))).t()
        gb[e] = g.t() @ u
        gbe[e] = g.abs().t() @ (ue + (n + 8) * U * (u.abs() + ue))
    fin = lambda v, e: (v, e + h * (v.abs() + e) + tiny)  # noqa: E731
    return fin(out, oe + 2 * U * out.abs()), fin(gx, gxe), fin(ga, gae), fin(gb, gbe)


def within(got, want, what):
    v, e = want
    off = (got.double().cpu() - v).abs()
    assert got.shape == v.shape
    worst = (off / e.clamp(min=1e-300)).max() if off.numel() else 0.0
    assert bool((off <= e).all()), (what, float(worst))


def run(d, ids=True, check=True, **kw):
    dev = {k: v.to(DEV) for k, v in d.items()}
    x, a, b, base = (dev[k].requires_grad_() for k in ("x", "a", "b", "base"))
    out = lora_add(base, x, a, b, adapter_ids=dev["ids"] if ids else None, scaling=dev["s"],
                   check_status=check, **kw)
    grads = torch.autograd.grad(out, [x, a, b, base], dev["g"])
    return (out.detach(), *grads)


def check(d, dtype, ids=True):
    got = run(d, ids)
    names = ("out", "x's gradient", "a's", "b's")
    for t, w, name in zip(got, expect(d, dtype), names):
        assert t.dtype == dtype
        within(t, w, name)
    assert torch.equal(got[4].cpu(), d["g"])
    # rows without an adapter are base's, to the bit
    none = d["ids"] == -1
    assert torch.equal(got[0].cpu()[none], d["base"][none])
    assert not got[1].cpu()[none].any()
    with torch.no_grad():
        dev = {k: v.to(DEV) for k, v in d.items()}
        again = lora_add(dev["base"], dev["x"], dev["a"], dev["b"],
                         adapter_ids=dev["ids"] if ids else None, scaling=dev["s"],
                         check_status=False)
    assert torch.equal(again, got[0])


@pytest.mark.parametrize("dtype", [BF, HF, F4], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,S,K,N,E,r", [
    (1, 1, 1, 1, 1, 1), (1, 1, 64, 64, 1, 16), (3, 1, 65, 33, 2, 8), (5, 7, 128, 96, 3, 4),
    (2, 17, 1027, 515, 2, 5), (64, 1, 512, 704, 8, 16), (200, 1, 96, 130, 40, 24),
    (4, 100, 256, 1030, 3, 32), (3, 500, 200, 72, 2, 64), (7, 300, 136, 264, 5, 8),
    (2, 700, 64, 48, 2, 100), (1, 1500, 520, 1000, 1, 16), (2, 30, 80, 40, 2, 256),
    (2, 700, 40, 56, 1, 256), (1025, 1, 24, 40, 1024, 8), (1, 3, 4096, 4096, 1, 16),
])
def test_rows_and_gradients(B, S, K, N, E, r, dtype):
    print("lora", B, S, K, N, E, r, dtype, flush=True)
    check(make(B, S, K, N, E, r, dtype, seed=K + r), dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F4], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,S,K,N,E,r", [
    (1, 2049, 520, 1000, 1, 128), (7, 300, 1027, 515, 3, 33), (90, 20, 136, 264, 5, 48),
    (1030, 1, 264, 136, 70, 40), (5, 411, 2048, 72, 2, 64),
])
def test_many_rows_of_larger_ranks(B, S, K, N, E, r, dtype):
    print("lora", B, S, K, N, E, r, dtype, flush=True)
    check(make(B, S, K, N, E, r, dtype, seed=K + r), dtype)


@pytest.mark.parametrize("dtype", [BF, F4], ids=["bf16", "fp32"])
@pytest.mark.parametrize("S", [1, 15, 64, 1024, 1025, 2049])
def test_one_adapter_for_all(S, dtype):
    d = make(1, S, 96, 160, 1, 16, dtype, seed=S, none=0.0)
    check(d, dtype, ids=False)
    # its adapters without their dimension, one number for the scale
    dev = {k: v.to(DEV) for k, v in d.items()}
    a, b = dev["a"][0].requires_grad_(), dev["b"][0].requires_grad_()
    out = lora_add(dev["base"][0], dev["x"][0], a, b, scaling=float(d["s"][0]))
    want = run(d)
    assert torch.equal(out, want[0][0])
    for got, w in zip(torch.autograd.grad(out, [a, b], dev["g"][0]), want[2:4]):
        assert torch.equal(got, w[0])


@pytest.mark.parametrize("kind", ["none", "one of many", "sorted", "falling", "last"])
def test_ids_of_every_kind(kind):
    for B, S in ((40, 1), (6, 250), (130, 16)):
        d = make(B, S, 64, 72, 9, 8, BF, seed=B)
        d["ids"] = {"none": torch.full((B,), -1), "one of many": torch.full((B,), 4),
                    "sorted": torch.arange(B) * 9 // B, "falling": 8 - torch.arange(B) * 9 // B,
                    "last": torch.full((B,), 8)}[kind]
        check(d, BF)
        d["ids"] = d["ids"].int()
        check(d, BF)


def test_an_id_for_each_row():
    d = make(6, 1, 64, 72, 3, 8, BF, seed=1)
    per_row = torch.tensor([[0, 2], [1, -1], [2, 2]])
    dev = {k: v.to(DEV) for k, v in d.items()}
    flat = lora_add(dev["base"], dev["x"], dev["a"], dev["b"],
                    adapter_ids=per_row.reshape(6).to(DEV), scaling=dev["s"])
    rows = lora_add(dev["base"].view(3, 2, -1), dev["x"].view(3, 2, -1), dev["a"], dev["b"],
                    adapter_ids=per_row.to(DEV), scaling=dev["s"])
    assert torch.equal(flat.flatten(), rows.flatten())


def test_bad_ids():
    d = make(6, 5, 64, 72, 3, 8, BF, seed=2, none=0.0)
    good = run(d)
    d["ids"][2], d["ids"][4] = 3, -2
    with pytest.raises(RuntimeError, match="adapter id"):
        run(d)
    d["ids"][2] = 2 ** 40 + 1
    with pytest.raises(RuntimeError, match="adapter id"):
        run(d)
    got = run(d, check=False)
    bad = torch.tensor([2, 4])
    ok = torch.tensor([0, 1, 3, 5])
    assert got[0][bad].isnan().all() and got[1][bad].isnan().all()
    assert torch.equal(got[0][ok], good[0][ok]) and torch.equal(got[1][ok], good[1][ok])
    d["ids"][bad] = -1
    for a, b in zip(got[2:4], run(d)[2:4]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F4], ids=["bf16", "fp32"])
def test_layouts(dtype):
    d = make(3, 70, 66, 90, 2, 8, dtype, seed=3)
    want = run(d)
    dev = {k: v.to(DEV) for k, v in d.items()}

    def odd(t, pad):
        """The same values, rows apart, from an odd element on."""
        flat = torch.zeros(t.numel() // t.shape[-1] * (t.shape[-1] + pad) + 1, dtype=t.dtype,
                           device=DEV)
        v = flat[1:].view(-1, t.shape[-1] + pad)[:, : t.shape[-1]]
        v.copy_(t.reshape(-1, t.shape[-1]))
        return v.view(*t.shape[:-1], -1) if t.dim() < 3 else flat[1:].view(
            *t.shape[:-1], t.shape[-1] + pad)[..., : t.shape[-1]]

    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    columns = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    for f in (lambda t: odd(t, 3), turned, columns):
        v = {k: f(dev[k]).requires_grad_() for k in ("base", "x", "a", "b")}
        out = lora_add(v["base"], v["x"], v["a"], v["b"], adapter_ids=dev["ids"], scaling=dev["s"])
        grads = torch.autograd.grad(out, [v["x"], v["a"], v["b"]], f(dev["g"]))
        for a, b in zip((out, *grads), want):
            assert torch.equal(a, b)
    # a base and a gradient that are broadcast, x shared by the sequences
    one = dev["x"][:1, :1].expand_as(dev["x"]).detach().requires_grad_()
    out = lora_add(dev["base"][:1, :1].expand_as(dev["base"]), one, dev["a"], dev["b"],
                   adapter_ids=dev["ids"], scaling=dev["s"])
    gx, = torch.autograd.grad(out.sum(), [one])
    e = dict(d, x=d["x"][:1, :1].expand_as(d["x"]).contiguous(), g=torch.ones_like(d["g"]),
             base=d["base"][:1, :1].expand_as(d["base"]).contiguous())
    w = expect(e, dtype)
    within(out.detach(), w[0], "out")
    within(gx, w[1], "x's gradient")


def test_parts_of_the_gradients():
    d = make(3, 50, 66, 90, 2, 8, BF, seed=4)
    want = run(d)
    dev = {k: v.to(DEV) for k, v in d.items()}
    for need in range(1, 16):
        t = [dev[k].detach().clone().requires_grad_(bool(need >> i & 1))
             for i, k in enumerate(("x", "a", "b", "base"))]
        out = lora_add(t[3], t[0], t[1], t[2], adapter_ids=dev["ids"], scaling=dev["s"])
        out.backward(dev["g"])
        for i in range(4):
            if need >> i & 1:
                assert torch.equal(t[i].grad, want[1 + i])
            else:
                assert t[i].grad is None


def test_values_where_the_low_part_matters():
    # outputs without a base, from low-rank values that 16 bits round
    for dtype in (BF, HF):
        d = make(2, 40, 300, 64, 1, 16, dtype, seed=5, none=0.0)
        d["base"].zero_()
        d["ids"].zero_()
        check(d, dtype)
        got = run(d)[0].cpu().double()
        v = expect(d, dtype)[0][0]
        # the output's own rounding and hardly more: rounding U alone would add as much again
        rel = float((got - v).norm() / v.norm())
        assert rel < 0.45 * torch.finfo(dtype).eps, rel


def test_low_rank_values_past_fp16s_range():
    """u above 65504 with b that brings it back, v far below 2^-14: the parts are
    bf16's, so neither is lost."""
    for up, down, grad in ((2.0 ** 12, 2.0 ** -14, 2.0 ** -4), (2.0 ** -8, 2.0 ** -12, 2.0 ** -6)):
        d = make(2, 200, 256, 64, 1, 16, HF, seed=31, none=0.0)
        d["ids"].zero_()
        d["base"].zero_()
        d["a"] = (d["a"].double() * up).to(HF)
        d["b"] = (d["b"].double() * down).to(HF)
        d["g"] = (d["g"].double() * grad).to(HF)
        check(d, HF)
        want = expect(d, HF)
        u = (d["x"][0].double() @ d["a"][0].double().t()).abs().max()
        v = (d["g"][0].double() @ d["b"][0].double()).abs().median()
        assert u > 65504 or v < 2.0 ** -13
        for got, (w, _), name in zip(run(d), want, ("out", "gx", "ga", "gb")):
            # as far as the values themselves are normal numbers: one rounding of
            # them, and 2^-16 of what is summed
            ok = w.abs() > 2.0 ** -13
            if ok.any():
                rel = float((got.double().cpu() - w)[ok].norm() / w[ok].norm())
                assert rel < 2.0 ** -11, (name, rel)


def test_infinities_and_nan_stay_in_their_rows():
    d = make(4, 20, 64, 72, 2, 8, BF, seed=6, none=0.0)
    clean = run(d)
    d["x"][1, 3, 5] = float("inf")
    d["x"][2, 7, 0] = float("nan")
    d["base"][3, 1, 2] = float("inf")
    got = run(d)
    hurt = torch.zeros(4, 20, dtype=torch.bool)
    hurt[1, 3] = hurt[2, 7] = hurt[3, 1] = True
    assert torch.equal(got[0].cpu()[~hurt], clean[0].cpu()[~hurt])
    assert not got[0].cpu()[1, 3].isfinite().any() and got[0].cpu()[2, 7].isnan().all()
    assert got[0][3, 1, 2] == float("inf") and torch.equal(got[1], clean[1])


def test_no_rows():
    a, b = torch.zeros(2, 4, 8, device=DEV, requires_grad=True), torch.zeros(2, 6, 4, device=DEV)
    for shape in ((0, 5), (3, 0), (0,)):
        ids = torch.zeros(shape[0], dtype=torch.int64, device=DEV)
        out = lora_add(torch.zeros(*shape, 6, device=DEV), torch.zeros(*shape, 8, device=DEV), a, b,
                       adapter_ids=ids)
        assert out.shape == (*shape, 6)
        ga, = torch.autograd.grad(out.sum(), [a])
        assert torch.equal(ga, torch.zeros_like(a))


def test_an_adapter_without_rows_has_zeros():
    d = make(3, 30, 64, 72, 6, 8, BF, seed=7, none=0.0)
    d["ids"] = torch.tensor([1, 4, 4])
    got = run(d)
    for e in (0, 2, 3, 5):
        assert not got[2][e].any() and not got[3][e].any()


def test_the_same_bits_every_time():
    d = make(9, 211, 520, 264, 4, 16, BF, seed=8)
    first = run(d)
    for _ in range(3):
        for a, b in zip(first, run(d)):
            assert torch.equal(a, b)


def test_twice_backwards_raises():
    d = make(1, 4, 16, 16, 1, 4, F4, seed=9, none=0.0)
    dev = {k: v.to(DEV) for k, v in d.items()}
    x = dev["x"].requires_grad_()
    out = lora_add(dev["base"], x, dev["a"], dev["b"], adapter_ids=dev["ids"])
    gx, = torch.autograd.grad(out.square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        gx.sum().backward()
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        lora_add(dev["base"], fwAD.make_dual(dev["x"].detach(), dev["x"].detach()), dev["a"],
                 dev["b"], adapter_ids=dev["ids"])


def test_gradients_against_differences():
    d = make(2, 3, 12, 10, 2, 3, F4, seed=10, none=0.0)
    dev = {k: v.to(DEV) for k, v in d.items()}
    f = lambda x, a, b: float((lora_add(dev["base"], x, a, b, adapter_ids=dev["ids"],  # noqa: E731
                                        scaling=dev["s"]).double() * dev["g"]).sum())
    got = run(d)
    args = [dev["x"], dev["a"], dev["b"]]
    for i, grad in enumerate(got[1:4]):
        direction = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        eps = 2.0 ** -6  # (the output is linear in each operand: no higher terms)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * direction, args[i] - eps * direction
        want = (f(*up) - f(*down)) / (2 * eps)
        size = float((grad.double().abs() * direction.abs()).sum())
        # two evaluations of sums of below 2^8 fp32 products, over 2 eps
        assert abs(float((grad.double() * direction).sum()) - want) < size * 2.0 ** -10


def test_captured_and_replayed():
    d = make(5, 60, 128, 96, 3, 8, BF, seed=11)
    dev = {k: v.to(DEV) for k, v in d.items()}
    x, a, b = (dev[k].requires_grad_() for k in ("x", "a", "b"))

    def step():
        out = lora_add(dev["base"], x, a, b, adapter_ids=dev["ids"], scaling=dev["s"])
        return (out, *torch.autograd.grad(out, [x, a, b], dev["g"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        new = make(5, 60, 128, 96, 3, 8, BF, seed=20 + i)
        with torch.no_grad():
            for k in d:
                dev[k].copy_(new[k])
        want = run(new)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for got, w in zip(out, want):
                assert torch.equal(got, w), i


def test_a_capture_beside_an_eager_graph_is_refused():
    d = make(1, 4, 16, 16, 1, 4, BF, seed=12, none=0.0)
    dev = {k: v.to(DEV) for k, v in d.items()}
    for dim in (3, 2):
        a = dev["a"].detach().clone()
        b = dev["b"]
        if dim == 2:
            a, b = a[0].clone(), b[0]
        a.requires_grad_()
        alive = lora_add(dev["base"], dev["x"], a, b)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph):
                lora_add(dev["base"], dev["x"], a, b)
        del alive


def test_another_stream():
    d = make(5, 60, 128, 96, 3, 8, BF, seed=13)
    want = run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(d)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_the_scaling_and_the_ids_may_be_refilled():
    d = make(5, 20, 32, 24, 3, 8, BF, seed=14)
    want = run(d)
    dev = {k: v.to(DEV) for k, v in d.items()}
    x, a, b = (dev[k].requires_grad_() for k in ("x", "a", "b"))
    out = lora_add(dev["base"], x, a, b, adapter_ids=dev["ids"], scaling=dev["s"])
    dev["s"].zero_()
    dev["ids"].fill_(0)
    for got, w in zip(torch.autograd.grad(out, [x, a, b], dev["g"]), want[1:]):
        assert torch.equal(got, w)


def test_rows_past_32_bit_offsets():
    # x's rows lie 2^30 elements apart
    d = make(3, 1, 64, 72, 2, 8, BF, seed=15, none=0.0)
    dev = {k: v.to(DEV) for k, v in d.items()}
    far = torch.zeros(3, (1 << 30) + 8, dtype=BF, device=DEV)
    far[:, :64].copy_(dev["x"][:, 0])
    x = far[:, :64].unsqueeze(1)
    out = lora_add(dev["base"], x, dev["a"], dev["b"], adapter_ids=dev["ids"], scaling=dev["s"])
    assert torch.equal(out, run(d)[0])


def test_the_state_of_other_sizes_is_refused():
    d = make(3, 5, 64, 72, 2, 8, BF, seed=16)
    dev = {k: v.to(DEV) for k, v in d.items()}
    out, state = ops.lora_add_state(dev["base"], dev["x"], dev["a"], dev["b"],
                                    adapter_ids=dev["ids"], scales=dev["s"])
    assert torch.equal(out, run(d)[0])
    with pytest.raises(RuntimeError, match="state"):
        ops.lora_backward(dev["g"], dev["x"], dev["a"], dev["b"], state[:-256], requests=3)
    gx, ga, gb = ops.lora_backward(dev["g"], dev["x"], dev["a"], dev["b"], state, requests=3,
                                   need_a=False)
    want = run(d)
    assert torch.equal(gx, want[1]) and ga is None and torch.equal(gb, want[3])
