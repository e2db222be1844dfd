"""What the two public forms of the losses from hidden states,
``graspo_loss.sequence_log_probs_from_hidden`` and
``sft_loss.sft_cross_entropy_loss_from_hidden``, check alike."""

from __future__ import annotations

import torch


def check_operands(what: str, hidden: torch.Tensor, weight: torch.Tensor) -> None:
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: expected hidden states [..., K] and a weight [V, K], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden states and weight must both be bfloat16 or both float16, "
                         f"got {hidden.dtype} and {weight.dtype}")
