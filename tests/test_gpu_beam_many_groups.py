"""A beam step of more groups than one dimension of a launch holds: the merge has a
workgroup of 1024 threads for each.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.beam_search import beam_start, beam_step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16


def test_a_step_of_many_groups():
    """2^22 groups of the merge's 1024 threads."""
    G, V = (1 << 22) + 3, 5
    print("beam step", G, flush=True)
    row = torch.arange(G, device=DEV).unsqueeze(1)
    x = ((3 * torch.arange(V, device=DEV) + row) % 7).to(BF)  # distinct in a row
    scores = -(row % 11).float()
    c = (scores.double() + torch.log_softmax(x.double(), -1)).sort(descending=True)
    # 5 exponentials, each off by 2^-23, their sum and one rounding; |c| < 18
    off = (5 + 4) * 2.0 ** -23 + 18 * 2.0 ** -24
    got = ops.beam_candidates(x, scores, candidates=2)
    assert torch.equal(got.tokens, c.indices[:, :2]) and not got.beams.any()
    assert (got.scores.double() - c.values[:, :2]).abs().max() <= off and not got.status.any()
    state = beam_start(G, 1, DEV)._replace(scores=scores)
    step = beam_step(x, state, eos_token_id=V + 1, pad_token_id=0)
    assert torch.equal(step.tokens, c.indices[:, 0])
    assert torch.equal(step.parents, row[:, 0].int())
    assert torch.equal(step.state.scores, got.scores[:, :1]) and not step.state.done.any()
