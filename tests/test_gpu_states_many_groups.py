"""States of more than 2^32 - 1 work items, which one dimension of a launch does not
hold: many groups of short rows, long rows of an odd number of bytes.  Whole bytes
moved, so every comparison is exact.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd.beam_search import expand_states, reorder_states_

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("K", [2, 17])
def test_states_of_many_groups(K):
    """2^24 workgroups of 256."""
    G = (1 << 24) + 5
    print("states", G, K, flush=True)
    R = G * K
    t = (torch.arange(R, dtype=torch.int32, device=DEV) * 40503 >> 7).to(torch.uint8).unsqueeze(1)
    row = torch.arange(R, dtype=torch.int32, device=DEV)
    parents = row - row % K + (row % K + 1 + row // K % 2) % K
    want = t[parents.long()]
    reorder_states_([t], parents, K)
    assert torch.equal(t, want)


def test_copies_of_many_groups():
    G = (1 << 24) + 5
    print("copies", G, flush=True)
    t = (torch.arange(G, dtype=torch.int32, device=DEV) * 40503 >> 7).to(torch.uint8).unsqueeze(1)
    got, = expand_states([t], 2)
    assert torch.equal(got, t.repeat_interleave(2, 0))


def test_states_with_a_row_of_many_units():
    """Rows of an odd number of bytes, 2^23 workgroups each, in a launch of 3."""
    G, K, n = 3, 2, (1 << 31) - 255
    print("long rows", flush=True)
    t = torch.empty((G * K, n), dtype=torch.uint8, device=DEV)
    ends = torch.arange(G * K * 64, device=DEV).to(torch.uint8).view(G * K, 64)
    for at in (0, n // 2, n - 64):
        t[:, at:at + 64] = ends + at % 251
    parents = torch.tensor([1, 0, 2, 2, 5, 4], device=DEV)
    reorder_states_([t], parents, K)
    for at in (0, n // 2, n - 64):
        assert torch.equal(t[:, at:at + 64], (ends + at % 251)[parents])
