"""A vocabulary row of -inf logits at every number of rows that take part.

Its own gradient is sum_n D_n h_n with D = 0 for every token, so exactly 0.
The gradients of the others are those without it; tolerances are expect()'s.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd.graspo_loss import sequence_log_probs_from_hidden
from test_gpu_linear_logprob import expect, inputs, within

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("value", [float("-inf"), float("nan")])
@pytest.mark.parametrize("N,drop", [(5, 0), (70, 3), (129, 0), (130, 0), (136, 0), (261, 0),
                                    (261, 5), (300, 171), (520, 7), (140, 139)])
def test_rows_past_the_last_make_no_nan(N, drop, value, dtype):
    """`drop` of the rows have gradient 0, so that the number of those that
    take part is a multiple of 8 or not, and of 256 or not.  NaN, in the column
    that every hidden state has at 0: 0 * NaN is a NaN logit for every token,
    and the whole weight's gradient with it."""
    V, K = 40, 64
    h, w, t, g = inputs(N, V, K, dtype, seed=N)
    g = g.abs() + 0.125
    g[torch.randperm(N, generator=torch.Generator().manual_seed(drop))[:drop]] = 0.0
    h = h.abs() + 0.5
    w[7], w[7, 3] = 0.0, value
    t[t == 7] = 8
    hd, wd = h.cuda(), w.cuda().requires_grad_()
    got = sequence_log_probs_from_hidden(hd, wd, t.cuda())
    (gw,) = torch.autograd.grad(got, [wd], g.cuda())
    if value != value:
        assert bool(got.isnan().all()) and bool(gw.isnan().all())
        return
    keep = torch.arange(V) != 7
    small = torch.where(t > 7, t - 1, t)
    lp, lp_e, _, _, want, err = expect(h, w[keep], small, g, dtype)
    within(got.detach().cpu(), lp, lp_e, "logprob")
    assert bool((gw[7] == 0).all())
    within(gw.cpu()[keep], want, err, "weight's gradient")
