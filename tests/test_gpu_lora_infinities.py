"""Infinities and the largest numbers in adapters' operands: where the formula,
in the operands' order of products, gives an infinity, so do the kernels, and
NaN only where it does.  u and v as two 16-bit parts must not make one of the
other."""

from __future__ import annotations

import pytest
import torch

from graspo_amd.lora import lora_add

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")
TYPES = pytest.mark.parametrize("dtype", [BF, HF, F4], ids=["bf16", "fp16", "fp32"])


def product(x, w):
    """x w, every product on its own: an infinity beside zeros is not NaN."""
    return (x.unsqueeze(-1) * w.unsqueeze(-3)).sum(-2)


def formula(d):
    x, a, b, base, g = (d[k].double() for k in ("x", "a", "b", "base", "g"))
    u, v = product(x, a.t()), product(g, b)
    return (base + product(u, b.t()), product(v, a), product(v.t(), x), product(g.t(), u))


def run(d):
    dev = {k: v.to(DEV) for k, v in d.items()}
    x, a, b = (dev[k].requires_grad_() for k in ("x", "a", "b"))
    out = lora_add(dev["base"], x, a, b)
    return [t.detach().cpu() for t in (out, *torch.autograd.grad(out, [x, a, b], dev["g"]))]


def make(rows, K, N, r, dtype, seed, positive=False):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s):
        # no zeros among them, powers of two that need one part only, and no sum
        # of 1500 that leaves fp16
        t = (torch.randn(*s, generator=g) / 4).to(dtype)
        one = torch.full_like(t, 0.25)
        t = torch.where(torch.rand(*s, generator=g) < 0.3, one.copysign(t), t)
        t = torch.where(t == 0, one, t)
        return t.abs() if positive else t

    return dict(x=rnd(rows, K), a=rnd(r, K), b=rnd(N, r), base=rnd(rows, N), g=rnd(rows, N))


def compare(d, clean):
    """The same infinities and NaN as the formula's; what is finite, to the bit
    what it is without them."""
    got, plain = run(d), run(clean)
    hit = 0
    for t, p, w, name in zip(got, plain, formula(d), ("out", "x's", "a's", "b's")):
        assert torch.equal(t.isnan(), w.isnan()), name
        for inf in (INF, -INF):
            assert torch.equal(t == inf, w == inf), name
        fine = w.isfinite()
        assert torch.equal(t[fine], p[fine]), name
        hit += int((~fine).sum())
    assert hit > 0


@TYPES
@pytest.mark.parametrize("rows", [1, 40, 1500])
@pytest.mark.parametrize("name", ["x", "a", "b", "g"])
@pytest.mark.parametrize("r,positive", [(1, False), (5, True), (40, True)])
def test_an_infinity(name, rows, r, positive, dtype):
    print("infinity in", name, rows, r, dtype, flush=True)
    clean = make(rows, 70, 36, r, dtype, seed=rows + r, positive=positive)
    for inf in (INF, -INF):
        d = dict(clean, **{name: clean[name].clone()})
        d[name][-1, 0] = inf
        compare(d, clean)


@TYPES
def test_infinities_of_both_signs(dtype):
    # inf - inf in u, v and the products
    clean = make(40, 70, 36, 5, dtype, seed=1)
    for name in ("x", "a", "b", "g"):
        d = dict(clean, **{name: clean[name].clone()})
        d[name][0, 0], d[name][0, 1], d[name][1, 2] = INF, -INF, INF
        compare(d, clean)


@pytest.mark.parametrize("dtype", [BF, F4], ids=["bf16", "fp32"])
def test_low_rank_values_near_the_largest(dtype):
    """u = 2^127 (2 - 2^-8), which bf16's nearest would make an infinity."""
    x = torch.full((3, 9), 2.0 ** 100, dtype=dtype)
    a = (2.0 ** (27.0 - torch.arange(9))).unsqueeze(0).to(dtype)
    b = torch.full((20, 1), 2.0 ** -100, dtype=dtype)
    base = torch.zeros(3, 20, dtype=dtype)
    for sign in (1.0, -1.0):
        got = lora_add(base.to(DEV), (sign * x).to(DEV), a.to(DEV), b.to(DEV)).cpu().double()
        want = sign * 2.0 ** 27 * (2 - 2.0 ** -8)
        # two parts hold it whole, and the output is rounded once
        assert (got - want).abs().max() <= torch.finfo(dtype).eps / 2 * abs(want)
