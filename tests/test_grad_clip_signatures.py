"""The clipping takes what torch.nn.utils' functions of the same names take."""

import inspect

import pytest
import torch

from graspo_amd import grad_clip


@pytest.mark.parametrize("name", ["get_total_norm", "clip_grads_with_norm_", "clip_grad_norm_"])
def test_same_arguments(name):
    theirs = inspect.signature(getattr(torch.nn.utils, name)).parameters
    ours = inspect.signature(getattr(grad_clip, name)).parameters
    assert list(ours) == list(theirs)
    assert [p.default for p in ours.values()] == [p.default for p in theirs.values()]


@pytest.mark.parametrize("foreach", [None, True, False])
def test_foreach_says_nothing_here(foreach):
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(grad_clip.clip_grad_norm_([p], 1.0, foreach=foreach)) == 0.0
    assert float(grad_clip.get_total_norm([], foreach=foreach)) == 0.0
    assert grad_clip.clip_grads_with_norm_([p], 1.0, torch.tensor(1.0), foreach=foreach) is None
