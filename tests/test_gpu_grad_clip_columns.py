"""Gradients that share memory without sharing an element: columns of one
buffer, as the parts of a fused projection's gradient are.  Tolerances are
those of test_gpu_grad_clip."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from graspo_amd.grad_clip import clip_grad_norm_, clip_grads_with_norm_
from test_gpu_grad_clip import W, check_clipped, exact_norm

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def parts(which, dtype):
    """(buffer, views that do not overlap, whether they leave elements out)."""
    g = torch.Generator().manual_seed(len(which))
    x = torch.randn(60, 96, generator=g).to(dtype).cuda()
    if which == "columns":
        return x, [x[:, :40], x[:, 40:56], x[:, 56:]], False
    if which == "columns out of order":
        return x, [x[:, 57:], x[:, 3:40], x[:, 40:57]], True
    if which == "every other row and column":
        return x, [x[::2, 1:50], x[1::2, 1:50], x[::2, 50:], x[1::2, 50:]], True
    if which == "blocks":
        return x, [x[:30, :40], x[30:, :90], x[:30, 40:90], x[:, 90:]], False
    if which == "even and odd elements":
        return x, [x.view(-1)[::2], x.view(-1)[1::2]], False
    if which == "transposed":
        return x, [x.t()[:40], x.t()[40:]], False
    if which == "a row among columns":
        return x, [x[:20, :40], x[:20, 40:], x[20], x[21:, 40:], x[21:, :40]], False
    cube = x.view(6, 10, 96)  # "heads"
    return x, [cube[:, :4, :48], cube[:, :4, 48:], cube[:, 4:]], False


ALL = ["columns", "columns out of order", "every other row and column", "blocks",
       "even and odd elements", "transposed", "a row among columns", "heads"]


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("which", ALL)
def test_parts_of_one_buffer(which, dtype):
    x, views, some_left = parts(which, dtype)
    before, whole = [v.cpu().clone() for v in views], x.cpu().clone()
    norm = exact_norm(before, 2)
    got = clip_grad_norm_([SimpleNamespace(grad=v) for v in views], 0.5 * norm)
    assert abs(float(got) - norm) <= (W + 1e-9) * norm
    check_clipped(views, before, norm, 0.5 * norm)
    # what no view shows is as it was
    for v in views:
        v.zero_()
    left = x.cpu() != 0
    assert bool(left.any()) == some_left and torch.equal(x.cpu()[left], whole[left])
    x.copy_(whole)
    clip_grads_with_norm_([SimpleNamespace(grad=v) for v in views], 0.5 * norm, got)
    check_clipped(views, before, norm, 0.5 * norm)


@pytest.mark.parametrize("which", ["one column twice", "columns that share one", "a block in columns",
                                   "a row through columns", "rows of other lengths",
                                   "an element among every other"])
def test_parts_that_share_an_element_are_refused(which):
    x = torch.randn(60, 96, device="cuda")
    keep = x.clone()
    flat = x.view(-1)
    views = {
        "one column twice": [x[:, :40], x[:, :40]],
        "columns that share one": [x[:, :40], x[:, 39:]],
        "a block in columns": [x[:, 40:], x[30:40, 50:60]],
        "a row through columns": [x[:, :40], x[:, 40:], x[7]],
        "rows of other lengths": [x[:, :40], flat[: 60 * 95].view(60, 95)[:, 40:]],
        "an element among every other": [flat[::2], flat[5 * 96 : 5 * 96 + 1]],
    }[which]
    for order in (views, views[::-1]):
        grads = [SimpleNamespace(grad=v) for v in order]
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grad_norm_(grads, 1e-3)
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads_with_norm_(grads, 1e-3, torch.tensor(1.0, device="cuda"))
    assert torch.equal(x, keep)
