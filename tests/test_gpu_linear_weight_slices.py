"""The lm_head's weight as the right part of a wider matrix, read in place: its
memory ends with its last row's last element.  The same bits as from a copy."""

from __future__ import annotations

import pytest
import torch

from graspo_amd.graspo_loss import sequence_log_probs_from_hidden
from test_gpu_linear_logprob import inputs

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N", [60, 300])
@pytest.mark.parametrize("V,K,wide", [(333, 192, 384), (256, 136, 272), (257, 320, 328), (700, 2880, 5760)])
def test_right_slices(V, K, wide, N, dtype):
    h, w, t, g = inputs(N, V, K, dtype, seed=V + K)
    big = torch.full((V, wide), float("nan"), dtype=dtype)
    big[:, wide - K:] = w
    right = big.cuda()[:, wide - K:]
    assert right.data_ptr() % 16 == 0
    outs = []
    for x in (right, w.cuda()):
        hd, x = h.cuda().requires_grad_(), x.detach().requires_grad_()
        lp = sequence_log_probs_from_hidden(hd, x, t.cuda())
        outs.append((lp.detach(), *torch.autograd.grad(lp, [hd, x], g.cuda())))
    for a, b in zip(*outs):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
