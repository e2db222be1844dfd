"""What is written in place counts as written: autograd's version counters
move, so that a graph that saved such a tensor raises instead of going on with
other values."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from graspo_amd import ops
from graspo_amd.grad_clip import clip_grad_norm_, clip_grads_with_norm_

pytestmark = pytest.mark.gpu


def params(*grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        out.append(p)
    return out


def gradients():
    gaps = torch.ones(6, 10, device="cuda")
    return [torch.ones(5, device="cuda"), torch.ones(3, 4, device="cuda").t(), gaps[:, :7],
            torch.ones(0, device="cuda")]


@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clipping_moves_the_versions(max_norm):
    """Where the factor is 1 too, as torch.nn.utils does."""
    norm = torch.tensor(2.0, device="cuda")
    for clip in (lambda p: clip_grad_norm_(p, max_norm),
                 lambda p: clip_grad_norm_(p, max_norm, error_if_nonfinite=True),
                 lambda p: clip_grads_with_norm_(p, max_norm, norm)):
        grads = gradients()
        before = [g._version for g in grads]
        clip(params(*grads))
        assert all(g._version > v for g, v in zip(grads, before))
        twin = gradients()
        torch.nn.utils.clip_grad_norm_(params(*twin), max_norm)
        assert all(t._version > 0 for t in twin if t.numel())
    assert norm._version == 0


def test_a_graph_over_a_clipped_gradient_raises():
    x = torch.randn(20, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), [x], create_graph=True)
    penalty = (g * g).sum()  # saves g
    p = torch.nn.Parameter(torch.zeros(20, device="cuda"))
    p.grad = g.detach()      # the same memory and counter
    clip_grad_norm_([p], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        penalty.backward()


def test_the_norm_alone_writes_nothing():
    grads = gradients()
    before = [g._version for g in grads]
    ops.grad_norm(grads)
    assert [g._version for g in grads] == before


def test_a_gradient_added_to_moves_its_version():
    ids = torch.tensor([1, 3, 1], device="cuda")
    to, grad = torch.zeros(5, 8, device="cuda"), torch.ones(3, 8, device="cuda")
    assert ops.embedding_backward(ids, grad, 5, out=to) is not None and to._version == 1
    order = ops.embedding_ordered(ids, to)[2]
    ops.embedding_backward(None, grad, 5, order=order, out=to)
    assert to._version == 2 and grad._version == 0 and order._version == 0
    # a tied gradient that a graph saved
    w = torch.randn(5, 8, device="cuda", requires_grad=True)
    y = (w * to).sum()
    ops.embedding_backward(ids, grad, 5, out=to)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_tensors_made_in_inference_mode():
    """They have no counter."""
    with torch.inference_mode():
        g, to = torch.ones(50, device="cuda"), torch.zeros(5, 8, device="cuda")
        norm = clip_grad_norm_([SimpleNamespace(grad=g)], 1.0)
        ops.embedding_backward(torch.tensor([1], device="cuda"), torch.ones(1, 8, device="cuda"), 5,
                               out=to)
    assert abs(float(norm) - 50 ** 0.5) < 1e-5 and bool((g < 1).all())
    assert float(to.sum()) == 8.0
