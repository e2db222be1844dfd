"""The embedding lookup, the vocabulary matrix's other end.

``token_embedding`` is ``F.embedding`` with a scale (models that multiply
their embeddings by sqrt(H) do it here, in fp32, rounded once).  Its gradient
sums the tokens' rows by sorted ids: the same bits on every run, where an
index_add's atomics give others.
"""

from __future__ import annotations

import torch

from . import ops


def token_embedding(
    input_ids: torch.Tensor,
    weight: torch.Tensor,
    *,
    scale: float = 1.0,
    padding_idx: int | None = None,
    check_status: bool = True,
) -> torch.Tensor:
    """``F.embedding(input_ids, weight, padding_idx) * scale``: [*ids, H] in
    the weight's dtype (fp32, bf16 or fp16), differentiable in ``weight``.  A
    negative ``padding_idx`` counts from the end; its row is looked up like
    any other and gets no gradient.  An id outside [0, V) raises
    ``RuntimeError``, for which the call waits for a look at the ids; with
    ``check_status=False`` (a decode loop, whose ids the sampler made), and in
    a graph capture, it does not wait, and such an id gives a row of NaN."""
    if weight.dim() != 2:
        raise ValueError(f"token_embedding: expected a weight [V, H], got {tuple(weight.shape)}")
    if weight.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"token_embedding: weight must be float32, bfloat16 or float16, got "
                         f"{weight.dtype}")
    if input_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"token_embedding: ids must be int32 or int64, got {input_ids.dtype}")
    V = weight.shape[0]
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"token_embedding: padding_idx {padding_idx} outside the table's {V} "
                             f"rows")
        padding_idx %= V
    return ops.token_embedding(input_ids, weight, scale=scale, padding_idx=padding_idx,
                               check=bool(check_status))
