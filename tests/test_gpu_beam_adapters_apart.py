"""A prompt under each adapter and under none gives different hypotheses, and
its logits are those of its own adapter alone."""

from __future__ import annotations

import builtins

import pytest
import torch

import test_gpu_beam_decode_loop as loop
from graspo_amd import decode_loop as dl
from graspo_amd.lora import lora_add
from test_gpu_requests_together import DEV, E, EOS, PAD, V, Adapter, AdapterLM

pytestmark = pytest.mark.gpu


def test_one_prompt_under_every_adapter():
    ids = torch.tensor([0, 1, 2, -1])
    assert len(ids) == E + 1
    prompt = torch.randint(8, V, (1, 4), generator=torch.Generator().manual_seed(0))
    args = dict(eos_token_id=EOS, pad_token_id=PAD, max_new_tokens=12, num_beams=4)
    out, scores, _ = dl.generate_beams_with_kv_cache(
        Adapter(AdapterLM(1, ids)), sequences=prompt.repeat(4, 1).to(DEV), **args)
    assert len({tuple(row) for row in out.tolist()}) == 4
    assert len(set(scores.flatten().tolist())) == 4


def test_logits_of_every_adapter():
    lm = AdapterLM(1, torch.tensor([0, 1, 2, -1]))
    g = torch.Generator().manual_seed(2)
    hidden = torch.randn(4, lm.a.shape[2], generator=g).to(torch.bfloat16).to(DEV)
    base = torch.nn.functional.linear(hidden, lm.head)
    got = lora_add(base, hidden, lm.a, lm.b, adapter_ids=lm.ids, scaling=0.5).double()
    u = 2.0 ** -24
    for i, e in enumerate(lm.ids.tolist()):
        want = base[i].double()
        if e >= 0:
            x, a, b = (t.double() for t in (hidden[i], lm.a[e], lm.b[e]))
            low = 0.5 * a @ x
            off = 0.5 * (72 * u) * (a.abs() @ x.abs()) + (2.0 ** -16 + 2 * u) * low.abs()
            off = b.abs() @ (off + 16 * u * (low.abs() + off))
            want = want + b @ low
            off = off + 2 * u * want.abs() + 2.0 ** -8 * (want.abs() + off)
            assert ((got[i] - want).abs() <= off).all()
            assert not torch.equal(got[i], base[i].double())
        else:
            assert torch.equal(got[i], want)


@pytest.mark.parametrize("args", [m for m in loop.test_search.pytestmark
                                  if m.name == "parametrize"][0].args[1], ids=str)
def test_no_near_ties_in_the_loops_searches(args, monkeypatch):
    """What the loop's own test takes for granted where a step has an exact tie:
    of scores that differ, none are nearer than 2e-5."""
    G, K, T, bias, penalty, early, give = args

    def least(values):
        values = list(values)
        apart = [v for v in values if v > 0]
        assert not apart or builtins.min(apart) > 2e-5
        return builtins.min(values)

    monkeypatch.setattr(loop, "min", least, raising=False)
    lm, p = loop.CacheLM(G * 100 + K, bias), loop.prompts(G, 5, seed=K)
    for g in range(G):
        loop.search(lm, p[g], K, T, penalty, early, give)
