"""Positions that take no part in a loss from hidden states keep out of its
gradients, whatever the loss's own gradient is.  Everything here is exact:
zeros, or NaN and infinities where the formula has them."""

from __future__ import annotations

import pytest
import torch

from graspo_amd.sft_loss import sft_cross_entropy_loss, sft_cross_entropy_loss_from_hidden

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
# (rows that a call has: up to 128, then more, then more than a tile)
SHAPES = [(2, 11), (1, 65), (4, 33), (2, 101), (3, 131)]


def step(B, S, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(B, S, 72, generator=g).to(dtype).cuda().requires_grad_()
    w = (torch.randn(300, 72, generator=g) / 8).to(dtype).cuda().requires_grad_()
    return h, w, torch.randint(0, 300, (B, S), generator=g).cuda()


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,S", SHAPES)
def test_a_mean_without_a_row_has_zero_gradients(B, S, dtype):
    """As F.cross_entropy: the loss is NaN, 0 / 0, its gradients are 0, so that
    a micro-batch of prompts alone leaves an accumulated gradient as it was."""
    h, w, _ = step(B, S, dtype)
    labels = torch.full((B, S), -100, device="cuda")
    for scale in (1.0, 0.125, 0.0):
        loss = sft_cross_entropy_loss_from_hidden(h, w, labels)
        assert bool(loss.isnan())
        for x in torch.autograd.grad(loss, [h, w], torch.tensor(scale, device="cuda")):
            assert bool((x == 0).all())
    held = torch.randn_like(w)
    w.grad = held.clone()
    sft_cross_entropy_loss_from_hidden(h, w, labels).backward()
    assert torch.equal(w.grad, held)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,S", SHAPES)
def test_ignored_positions_stay_zero_beside_a_gradient_that_is_not_finite(B, S, dtype):
    """A loss scale that overflows spoils the rows that take part, not the
    hidden states of those that do not: as the loss from logits has it."""
    h, w, labels = step(B, S, dtype)
    labels[:, S // 2:] = -100
    live = torch.zeros(B, S, dtype=torch.bool, device="cuda")
    live[:, :-1] = labels[:, 1:] != -100
    for v in (float("inf"), float("-inf"), float("nan")):
        g = torch.tensor(v, device="cuda")
        gh, gw = torch.autograd.grad(sft_cross_entropy_loss_from_hidden(h, w, labels), [h, w], g)
        assert bool((gh[~live] == 0).all())
        assert not bool(gh[live].isfinite().any()) and not bool(gw.isfinite().any())
        logits = (h.float() @ w.float().t()).detach().requires_grad_()
        (gx,) = torch.autograd.grad(sft_cross_entropy_loss(logits, labels), [logits], g)
        assert bool((gx[~live] == 0).all()) and not bool(gx[live].isfinite().any())
