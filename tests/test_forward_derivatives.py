"""Forward-mode derivatives (torch.func.jvp, dual tensors) of the operators that
are autograd nodes: refused, not dropped.  Without a GPU: the refusal comes
before anything else is looked at."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import graspo_amd

OPS = graspo_amd.load()
BF = torch.bfloat16


def logprobs(h, w):
    return OPS.linear_loss(h, w, torch.zeros(1, 5, dtype=torch.int64), None, False, "a loss", 0)


def mean(h, w):
    return OPS.linear_loss(h, w, torch.zeros(1, 4, dtype=torch.int64), -100, True, "a loss", 0)


def lookup(h, w):
    return OPS.token_embedding(torch.zeros(2, dtype=torch.int64), w, 1.0, -1, True, 0)


@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("call,which", [(logprobs, 0), (logprobs, 1), (mean, 0), (mean, 1), (lookup, 1)])
def test_dual_tensors_are_refused(call, which, needs_grad):
    args = [torch.zeros(1, 5, 16, dtype=BF), torch.zeros(9, 16, dtype=BF)]
    args[which].requires_grad_(needs_grad)
    with fw.dual_level():
        dual = list(args)
        dual[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(*dual)
        # tensors without a tangent go on (to there being no GPU)
        with pytest.raises(RuntimeError, match="GPU"):
            call(*args)
        # and so do duals where torch drops the tangents itself
        with torch.inference_mode(), pytest.raises(RuntimeError, match="GPU"):
            call(*dual)
    with pytest.raises(RuntimeError, match="GPU"):
        call(*args)


def test_jvp_is_refused():
    w = torch.zeros(9, 16, dtype=BF)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: lookup(None, x), (w,), (w,))
