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

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


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
    if x.dtype not in DTYPES:
        raise ValueError(f"lora_add: x must be float32, bfloat16 or float16, got {x.dtype}")
    for name, t in (("base", base), ("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dtype != x.dtype:
            raise ValueError(f"lora_add: {name} must be {x.dtype} as x, got {t.dtype}")
    if lora_a.dim() not in (2, 3) or lora_b.dim() != lora_a.dim():
        raise ValueError(f"lora_add: expected adapters [E, r, K] and [E, N, r] (or [r, K] and "
                         f"[N, r]), got {tuple(lora_a.shape)} and {tuple(lora_b.shape)}")
    E = lora_a.shape[0] if lora_a.dim() == 3 else 1
    (r, K), N = lora_a.shape[-2:], lora_b.shape[-2]
    if x.dim() < 1 or x.shape[-1] != K or lora_b.shape != (*lora_a.shape[:-2], N, r) or \
            base.shape != (*x.shape[:-1], N) or 0 in (E, r, K, N):
        raise ValueError(f"lora_add: base {tuple(base.shape)}, x {tuple(x.shape)} and adapters "
                         f"{tuple(lora_a.shape)}, {tuple(lora_b.shape)} do not go together")
    if r > 256 or E > 1024:
        raise ValueError(f"lora_add: at most 1024 adapters of rank 256, got {E} of {r}")
    if adapter_ids is None:
        if E != 1:
            raise ValueError(f"lora_add: {E} adapters and no adapter_ids")
    else:
        if adapter_ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lora_add: adapter_ids must be int32 or int64, got "
                             f"{adapter_ids.dtype}")
        if adapter_ids.dim() < 1 or adapter_ids.dim() >= x.dim() or \
                adapter_ids.shape != x.shape[:adapter_ids.dim()]:
            raise ValueError(f"lora_add: adapter_ids {tuple(adapter_ids.shape)} are not of the "
                             f"leading dimensions of x {tuple(x.shape)}")
        adapter_ids = adapter_ids.reshape(-1)
    scale, scales = 1.0, None
    if isinstance(scaling, torch.Tensor):
        if scaling.dtype != torch.float32 or scaling.shape != (E,):
            raise ValueError(f"lora_add: scaling must be a number or float32 [{E}], got "
                             f"{scaling.dtype} {tuple(scaling.shape)}")
        if scaling.requires_grad:
            raise ValueError("lora_add: the scaling has no gradient")
        scales = scaling.contiguous()
    else:
        scale = float(scaling)
    return ops.lora_add(base, x, lora_a, lora_b,
                        adapter_ids=None if adapter_ids is None else adapter_ids.contiguous(),
                        scales=scales, scale=scale, check=bool(check_status))
