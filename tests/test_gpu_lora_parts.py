"""Low-rank values as two bf16 parts, in fp16 too: hi is the value cut to 8
bits, lo what is left rounded to 8, off by 2^-16 of the value at most, over
fp32's range.  So the bounds have no absolute term but the results' own
rounding, and small gradients are held to the same relative error as large
ones.  (test_gpu_lora.py allows 2^-24 of each value in fp16 beside that, and
states 22 bits: neither what the kernels need nor what they hold.)"""

from __future__ import annotations

import pytest
import torch

from graspo_amd.lora import lora_add

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF = torch.bfloat16, torch.float16
U, PART = 2.0 ** -24, 2.0 ** -16


def within(got, want, size, off, terms, name):
    """Sums of `terms` fp32 products of absolute sum `size`, whose operands are
    off by `off` in all, and one rounding."""
    h, tiny = torch.finfo(got.dtype).eps / 2, 2.0 ** -24 if got.dtype == HF else 2.0 ** -133
    off = off + (terms + 8) * U * (size + off)
    off = off + h * (want.abs() + off) + tiny
    worst = ((got.double().cpu() - want).abs() / off).max()
    assert worst <= 1, (name, float(worst))


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows", [3, 300, 1500])
@pytest.mark.parametrize("up,down,grad", [(1.0, 1.0, 1.0), (2.0 ** 12, 2.0 ** -14, 2.0 ** -4),
                                          (1.0, 2.0 ** -12, 2.0 ** -10)])
def test_within_two_parts(rows, up, down, grad, dtype):
    print("parts", rows, up, down, grad, dtype, flush=True)
    K, N, r = 256, 72, 16
    g = torch.Generator().manual_seed(rows)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, a = rnd(rows, K).to(dtype), (rnd(r, K) * up / 16).to(dtype)
    b, go = (rnd(N, r) * down).to(dtype), (rnd(rows, N) * grad).to(dtype)
    base = torch.zeros(rows, N, dtype=dtype)
    dev = [t.to(DEV).requires_grad_() for t in (x, a, b)]
    out = lora_add(base.to(DEV), *dev)
    gx, ga, gb = torch.autograd.grad(out, dev, go.to(DEV))
    x, a, b, go = (t.double() for t in (x, a, b, go))
    u, v = x @ a.t(), go @ b
    ue = (K + 8) * U * (x.abs() @ a.t().abs()) + (PART + 2 * U) * u.abs()
    ve = (N + 8) * U * (go.abs() @ b.abs()) + (PART + 2 * U) * v.abs()
    within(out.detach(), u @ b.t(), u.abs() @ b.t().abs(), ue @ b.t().abs(), r, "out")
    within(gx, v @ a, v.abs() @ a.abs(), ve @ a.abs(), r, "x's gradient")
    within(ga, v.t() @ x, v.t().abs() @ x.abs(), ve.t() @ x.abs(), rows, "a's")
    within(gb, go.t() @ u, go.t().abs() @ u.abs(), go.t().abs() @ ue, rows, "b's")
