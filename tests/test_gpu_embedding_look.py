"""The look at the ids belongs to its call: one that raises for another reason
leaves nothing behind that answers for a later call."""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.embedding import token_embedding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ordered", [False, True])
def test_a_table_of_another_type_is_refused_ahead_of_the_look(ordered):
    call = ops.embedding_ordered if ordered else ops.embedding
    good, bad = torch.arange(9, device="cuda"), torch.full((9,), 99, device="cuda")
    table = torch.randn(20, 8, device="cuda")
    torch.cuda.synchronize()
    # (the look would wait here, and say "bad" after the call that made it)
    torch.cuda._sleep(1_000_000_000)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        call(bad, table.double())
    assert torch.equal(token_embedding(good, table), table[good])
    assert call(good, table)[1] is False and call(bad, table)[1] is True
