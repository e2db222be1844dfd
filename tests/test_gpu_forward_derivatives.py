"""Forward-mode derivatives of the losses from hidden states and the lookup, on
the GPU: refused in the forward, and in the backward of a gradient that has a
tangent."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from graspo_amd.embedding import token_embedding
from graspo_amd.graspo_loss import sequence_log_probs_from_hidden
from graspo_amd.sft_loss import sft_cross_entropy_loss_from_hidden

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def made():
    h = torch.randn(2, 5, 16, device="cuda").to(BF)
    return h, torch.randn(30, 16, device="cuda").to(BF), torch.arange(10, device="cuda").view(2, 5)


CALLS = {
    "logprobs": sequence_log_probs_from_hidden,
    "mean": sft_cross_entropy_loss_from_hidden,
    "lookup": lambda h, w, t: token_embedding(t, w),
}


@pytest.mark.parametrize("which", list(CALLS))
def test_tangents_of_the_operands(which):
    h, w, t = made()
    want = CALLS[which](h, w, t)
    with fw.dual_level():
        dual = fw.make_dual(w, torch.ones_like(w))
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[which](h, dual, t)
        if which != "lookup":
            with pytest.raises(RuntimeError, match="forward-mode"):
                CALLS[which](fw.make_dual(h, torch.ones_like(h)), w, t)
        assert torch.equal(CALLS[which](h, w, t), want)


@pytest.mark.parametrize("which", list(CALLS))
def test_tangents_of_the_gradient(which):
    h, w, t = made()
    w.requires_grad_()
    out = CALLS[which](h, w, t)
    (want,) = torch.autograd.grad(out, [w], torch.ones_like(out), retain_graph=True)
    with fw.dual_level():
        g = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, [w], g, retain_graph=True)
    assert torch.equal(torch.autograd.grad(out, [w], torch.ones_like(out))[0], want)
