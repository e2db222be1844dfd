"""Gradients that are part of a graph themselves (create_graph=True) are clipped
without being tracked, as torch.nn.utils does, whatever their layout.
Tolerances are those of test_gpu_grad_clip."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from graspo_amd.grad_clip import clip_grad_norm_, clip_grads_with_norm_
from test_gpu_grad_clip import W, check_clipped, exact_norm

pytestmark = pytest.mark.gpu


def layouts():
    base = torch.randn(6, 10, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    made = base * 2.0  # of a graph
    return {"a leaf": base, "a leaf's columns": base[:, :7], "made": made,
            "made's columns": made[:, 3:], "transposed": made.t()}


@pytest.mark.parametrize("which", ["a leaf", "a leaf's columns", "made", "made's columns",
                                   "transposed"])
def test_untracked(which):
    for by_norm in (False, True):
        g = layouts()[which]
        assert g.requires_grad
        before = [g.detach().cpu().clone()]
        norm, fn = exact_norm(before, 2), g.grad_fn
        if by_norm:
            clip_grads_with_norm_([SimpleNamespace(grad=g)], 0.5 * norm,
                                  torch.tensor(norm, dtype=torch.float32, device="cuda"))
        else:
            got = clip_grad_norm_([SimpleNamespace(grad=g)], 0.5 * norm)
            assert abs(float(got) - norm) <= (W + 1e-9) * norm and not got.requires_grad
        check_clipped([g.detach()], before, norm, 0.5 * norm)
        twin = layouts()[which]
        torch.nn.utils.clip_grads_with_norm_([SimpleNamespace(grad=twin)], 0.5 * norm,
                                             torch.tensor(norm, device="cuda"))
        # (a view written to names its node anew, untracked or not)
        assert type(g.grad_fn) is type(twin.grad_fn)
        assert (g.grad_fn is None) == (fn is None)
