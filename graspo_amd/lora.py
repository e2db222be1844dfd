"""Low-rank adapters beside a shared projection: a request's own, or none.

The reference's ``LoRALinear`` (``backends/graspoflow/lora.py:76``) adds one
adapter to a frozen projection, and training learns nothing else.
``lora_add`` is that addition for rows of many requests at once: what the
projection gave, plus each row's ``scaling (x A^T) B^T``, without a launch per
adapter or a product of the projection's size, and its gradients.
"""

from __future__ import annotations

import torch

from . import ops


def lora_add(
    base: torch.Tensor,
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    *,
    adapter_ids: torch.Tensor | None = None,
    scaling: float | torch.Tensor = 1.0,
    check_status: bool = True,
) -> torch.Tensor:
    """``base + scaling * (x @ A.T) @ B.T`` of each row's adapter, [..., N] in
    the operands' dtype (fp32, bf16 or fp16, all the same): ``x`` [..., K] is
    the projection's input, ``base`` [..., N] its output, ``lora_a`` [E, r, K]
    and ``lora_b`` [E, N, r] the adapters (r <= 256, E <= 1024), or [r, K] and
    [N, r] of a single one.  ``adapter_ids``, int32 or int64 of x's leading
    dimensions or the first of them (one id for all rows of a sequence), says
    which; -1 is none, such rows are base's.  ``scaling``: one number, or fp32
    [E] on the device (it has no gradient).

    Differentiable once, backwards, in base, x and the adapters.  Sums are fp32
    and the output is rounded once.  An id outside [-1, E) raises
    ``RuntimeError``, for which the call waits for a look at the ids; with
    ``check_status=False``, and in a graph capture, it does not wait, such rows
    are NaN and have no part in the adapters' gradients.
    """
    # (the op checks the arguments)
    if isinstance(scaling, torch.Tensor):
        return ops.lora_add(base, x, lora_a, lora_b, adapter_ids=adapter_ids, scales=scaling,
                            check=bool(check_status))
    return ops.lora_add(base, x, lora_a, lora_b, adapter_ids=adapter_ids, scale=float(scaling),
                        check=bool(check_status))
