"""early_stopping is a truth value: a word or a number is refused, for "never"
would be taken for True, its opposite.  Without a GPU."""

import numpy as np
import pytest
import torch

from graspo_amd import decode_loop as dl
from graspo_amd import ops
from graspo_amd.beam_search import beam_start, beam_step

BAD = ["never", "", 1, 0, 0.0, None, np.bool_(True), torch.tensor(True)]


@pytest.mark.parametrize("bad", BAD, ids=repr)
def test_refused(bad):
    state = beam_start(2, 3, "cpu")
    x = torch.zeros(6, 11)
    ids = dict(eos_token_id=1, pad_token_id=0)
    with pytest.raises(ValueError, match="early_stopping"):
        beam_step(x, state, early_stopping=bad, **ids)
    args = dict(length=1.0, step=0, early_stopping=bad, **ids)
    with pytest.raises(ValueError, match="early_stopping"):
        ops.beam_step(x, *state[:5], **args)
    c = ops.BeamCandidates(torch.zeros(2, 6), torch.zeros(2, 6).int(), torch.zeros(2, 6).long(),
                           torch.zeros(6).int())
    with pytest.raises(ValueError, match="early_stopping"):
        ops.beam_advance(c, *state[:5], **args)


class Model:
    def __init__(self):
        self.model = lambda *a, **k: pytest.fail("called")

    def _sync_timing(self):
        pass


@pytest.mark.parametrize("bad", BAD, ids=repr)
def test_the_loop_refuses_it_first(bad):
    prompt = torch.ones(1, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="early_stopping"):
        dl.generate_beams_with_kv_cache(Model(), sequences=prompt, eos_token_id=1, pad_token_id=0,
                                        max_new_tokens=3, num_beams=2, early_stopping=bad)
