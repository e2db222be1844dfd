"""Token logprobs and losses from hidden states and the lm_head weight.

What their two public forms, ``graspo_loss.sequence_log_probs_from_hidden`` and
``sft_loss.sft_cross_entropy_loss_from_hidden``, check alike.  Both are
:func:`graspo_amd.ops.linear_loss`: nothing of the size of the logits is kept
between forward and backward, which computes them again a piece of the
vocabulary at a time.  Against ``_selected_token_log_probs_from_hidden``
(tensor_utils.py), which keeps the fp32 logits: one product more, and 4 N V
bytes less (8.1 GB at 8192 tokens of 248320).
"""

from __future__ import annotations

import torch


def check_operands(what: str, hidden: torch.Tensor, weight: torch.Tensor) -> None:
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: expected hidden states [..., K] and a weight [V, K], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden states and weight must both be bfloat16 or both float16, "
                         f"got {hidden.dtype} and {weight.dtype}")
