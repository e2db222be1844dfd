"""Token logprobs and losses from hidden states and the lm_head weight.

The differentiable form of :func:`graspo_amd.ops.linear_logprob`: nothing of
the size of the logits is kept between forward and backward, which computes
them again a piece of the vocabulary at a time.  Against
``_selected_token_log_probs_from_hidden`` (tensor_utils.py), which keeps the
fp32 logits: one product more, and 4 N V bytes less (8.1 GB at 8192 tokens of
248320).  The public functions are
``graspo_loss.sequence_log_probs_from_hidden`` and
``sft_loss.sft_cross_entropy_loss_from_hidden``.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _LinearLogprob(torch.autograd.Function):
    """[B, T] logprobs, or their mean loss, of [B, S, K] hidden states."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, mean, what):
        out = ops.linear_logprob(hidden, weight, targets, ignore_index=ignore_index, mean=mean)
        if out.bad_target:
            raise RuntimeError(f"{what}: a target is outside [0, vocab_size)")
        grads = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        # a copy of the targets (8 bytes each): a loader may refill its labels
        # before the backward
        ctx.save_for_backward(hidden, weight, targets.clone() if grads else None, out.lse,
                              out.count if mean else None)
        ctx.ignore_index = ignore_index
        return out.mean_loss if mean else out.logprob

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, targets, lse, count = ctx.saved_tensors
        gh, gw = ops.linear_logprob_backward(
            hidden, weight, targets, lse, grad, mean_count=count, ignore_index=ctx.ignore_index,
            need_hidden=ctx.needs_input_grad[0], need_weight=ctx.needs_input_grad[1])
        return gh, gw, None, None, None, None


def check_operands(what: str, hidden: torch.Tensor, weight: torch.Tensor) -> None:
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: expected hidden states [..., K] and a weight [V, K], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden states and weight must both be bfloat16 or both float16, "
                         f"got {hidden.dtype} and {weight.dtype}")
