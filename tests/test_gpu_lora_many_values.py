"""Tables of adapters whose gradients take more than 2^32 - 1 work items, which one
dimension of a launch does not hold.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd.lora import lora_add

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16


def adapters(E, r, K, N, used):
    """Large tables of zeros but for the adapters in `used`."""
    g = torch.Generator().manual_seed(E + r)
    a = torch.zeros(E, r, K, dtype=BF, device=DEV)
    b = torch.zeros(E, N, r, dtype=BF, device=DEV)
    for e in used:
        a[e] = (torch.randn(r, K, generator=g) / K ** 0.5).to(BF)
        b[e] = torch.randn(N, r, generator=g).to(BF)
    x = torch.randn(len(used), 1, K, generator=g).to(BF).to(DEV)
    grad = torch.randn(len(used), 1, N, generator=g).to(BF).to(DEV)
    return a, b, x, grad


@pytest.mark.parametrize("E,r,K,N,need_x", [
    # 2^25 tiles of the table that the backward turns
    (1024, 1, (1 << 20) + 8, 3, True),
    # 2^32 values of the gradient and a few more
    (1024, 256, 16400, 2, False),
])
def test_adapters_of_many_values(E, r, K, N, need_x):
    print("adapters", E, r, K, N, flush=True)
    used = [E - 1, 0, E // 2]
    a, b, x, grad = adapters(E, r, K, N, used)
    a.requires_grad_()
    b.requires_grad_()
    x.requires_grad_(need_x)
    base = torch.zeros(len(used), 1, N, dtype=BF, device=DEV)
    out = lora_add(base, x, a, b, adapter_ids=torch.tensor(used, device=DEV))
    grads = torch.autograd.grad(out, [a, b] + ([x] if need_x else []), grad)
    U = 2.0 ** -24
    for i, e in enumerate(used):
        ad, bd = a[e].detach().double(), b[e].detach().double()
        xd, gd = x[i].detach().double(), grad[i].double()
        u, v = xd @ ad.t(), gd @ bd
        # 32-bit sums, two 16-bit parts, one rounding of the result
        ue = (K + 8) * U * (xd.abs() @ ad.t().abs()) + (2.0 ** -16 + 2 * U) * u.abs()
        ve = (N + 8) * U * (gd.abs() @ bd.abs()) + (2.0 ** -16 + 2 * U) * v.abs()
        rest = lambda w, y, e: e + (r + 8) * U * (y + e) + 2.0 ** -8 * (w.abs() + e)  # noqa: E731
        want = [(u @ bd.t(), u.abs() @ bd.t().abs(), ue @ bd.t().abs()),
                (v.t() @ xd, v.t().abs() @ xd.abs(), ve.t() @ xd.abs()),
                (gd.t() @ u, gd.t().abs() @ u.abs(), gd.t().abs() @ ue)]
        got = [out[i].detach(), grads[0][e], grads[1][e]]
        if need_x:
            want.append((v @ ad, v.abs() @ ad.abs(), ve @ ad.abs()))
            got.append(grads[2][i])
        for name, t, (w, y, err) in zip(("out", "a's", "b's", "x's"), got, want):
            assert ((t.double() - w).abs() <= rest(w, y, err)).all(), (e, name)
    # the others' gradients are zeros
    for t in grads[:2]:
        for lo, hi in ((1, E // 2), (E // 2 + 1, E - 1)):
            assert not t[lo:hi].any()
