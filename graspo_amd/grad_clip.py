"""The global gradient norm over many tensors, and clipping by it.

The names and arguments of ``torch.nn.utils``: one launch per 192 tensors for
the norm and one for the clipping, whatever their sizes and types, the norm
summed in 64 bits and the gradients rounded once (``foreach`` is torch's choice
between its own two ways, and says nothing here).  The reference's training
step clips between backward and optimizer
(``models/qwen35_36/training.py:427-441``).
"""

from __future__ import annotations

import torch

from . import ops


def _tensors(tensors) -> list[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _gradients(parameters) -> list[torch.Tensor]:
    return [g for p in _tensors(parameters) if (g := p.grad) is not None]


def _check(what: str, tensors: list[torch.Tensor], norm_type: float = 2.0) -> None:
    if norm_type not in (1.0, 2.0, float("inf")):
        raise ValueError(f"{what}: norm_type must be 1, 2 or inf, got {norm_type}")
    # (the op looks at each of a GPU's: a look from here takes 17 us for 504)
    if tensors and not tensors[0].is_cuda and any(t.is_sparse for t in tensors):
        raise ValueError(f"{what}: sparse gradients are not supported")


def _check_max_norm(what: str, max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must be at least 0, got {max_norm}")
    return max_norm


def _raise_if_nonfinite(what: str, norm: torch.Tensor, norm_type: float) -> None:
    if bool(norm.isnan()) or bool(norm.isinf()):
        raise RuntimeError(f"{what}: the total norm of order {norm_type} is non-finite, so the "
                           f"gradients cannot be clipped")


def get_total_norm(tensors, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                   foreach: bool | None = None) -> torch.Tensor:
    """The norm (``norm_type`` 1, 2 or inf) over all elements of ``tensors``
    (fp32, bf16, fp16, mixed, of one GPU) as an fp32 scalar on the device; 0
    without a tensor."""
    tensors = _tensors(tensors)
    norm_type = float(norm_type)
    _check("get_total_norm", tensors, norm_type)
    if not tensors:
        return torch.tensor(0.0)
    norm = ops.grad_norm(tensors, norm_type)
    if error_if_nonfinite:
        _raise_if_nonfinite("get_total_norm", norm, norm_type)
    return norm


def clip_grads_with_norm_(parameters, max_norm: float, total_norm: torch.Tensor,
                          foreach: bool | None = None) -> None:
    """Multiplies the parameters' gradients, in place, by min(1, ``max_norm``
    / (``total_norm`` + 1e-6)): ``total_norm`` as :func:`get_total_norm` gives
    it, or combined over ranks.  Gradients that overlap in memory (a parameter
    listed twice) raise ``RuntimeError``."""
    grads = _gradients(parameters)
    max_norm = _check_max_norm("clip_grads_with_norm_", max_norm)
    _check("clip_grads_with_norm_", grads)
    if grads:
        ops.clip_grads_(grads, total_norm.to(device=grads[0].device, dtype=torch.float32), max_norm)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """Clips the parameters' gradients, in place, to a total norm of
    ``max_norm`` and returns the norm that they had (an fp32 scalar on the
    device).  Without ``error_if_nonfinite`` nothing waits for the GPU; with
    it a norm that is NaN or infinite raises before any gradient is
    changed."""
    grads = _gradients(parameters)
    norm_type = float(norm_type)
    max_norm = _check_max_norm("clip_grad_norm_", max_norm)
    _check("clip_grad_norm_", grads, norm_type)
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = ops.grad_norm(grads, norm_type)
        _raise_if_nonfinite("clip_grad_norm_", norm, norm_type)
        ops.clip_grads_(grads, norm, max_norm)
        return norm
    return ops.clip_grad_norm_(grads, max_norm, norm_type)
