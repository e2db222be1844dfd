"""States of several shapes: where one cannot be moved, none is.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd.beam_search import reorder_states_

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_none_is_moved_where_one_is_refused():
    a = torch.arange(4, device=DEV).view(2, 2)
    # rows of more units than are supported: an odd number of bytes past 2^31
    b = torch.empty((2, (1 << 31) + 1), dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match="unsupported"):
        reorder_states_([a, b], torch.tensor([1, 0], device=DEV), 2)
    assert a.flatten().tolist() == [0, 1, 2, 3]
