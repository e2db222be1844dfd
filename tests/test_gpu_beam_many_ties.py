"""More equal scores than the merge compares with each other at once, and
hypotheses whose references lead nowhere: exact, by beam and token."""

from __future__ import annotations

import math

import pytest
import torch

from graspo_amd import ops
from graspo_amd.beam_search import beam_finish, beam_start, beam_step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32


def ranked(x, allowed, G, K, n):
    """(beam, token) of each group's n best, as if sorted stably: rows and
    scores are alike."""
    best = torch.sort(x.masked_fill(~allowed, -math.inf), descending=True, stable=True).indices[:n]
    c = sorted((-float(x[t]), k, int(t)) for k in range(K) for t in best)
    return [[(k, t) for _, k, t in c[:n]]] * G


@pytest.mark.parametrize("dtype", [BF, HF, F4], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("above", [0, 1, 2, 40])
@pytest.mark.parametrize("G,K,V,n", [(1, 32, 3000, 64), (2, 32, 20011, 64), (3, 20, 9000, 40),
                                     (1, 30, 150000, 60)])
def test_equal_rows(G, K, V, n, above, dtype):
    print("equal rows", G, K, V, n, above, dtype, flush=True)
    x = torch.zeros(V)
    x[torch.arange(above) * 71 + 5] = 1.0  # fewer of a row than are wanted, or none
    allowed = torch.ones(V, dtype=torch.bool)
    rows = x.to(dtype).to(DEV).expand(G, K, V)
    scores = torch.full((G, K), -3.0)
    got = ops.beam_candidates(rows, scores.to(DEV), candidates=n)
    want = ranked(x, allowed, G, K, n)
    assert [list(zip(b, t)) for b, t in zip(got.beams.tolist(), got.tokens.tolist())] == want
    lse = math.log(above * math.e + (V - above))
    exact = torch.tensor([[-3.0 + float(x[t]) - lse for _, t in w] for w in want],
                         dtype=torch.float64)
    # V exponentials, 256 steps of 2^-24 in all, and c's own rounding
    assert (got.scores.double().cpu() - exact).abs().max() <= 256 * 2.0 ** -24 + 32 * 2.0 ** -24
    assert not got.status.any()
    # with a mask, packed 32 tokens to a word
    allowed = torch.arange(V) % 3 != 1
    bits = torch.nn.functional.pad(allowed, (0, -V % 32)).view(-1, 32).long() << torch.arange(32)
    words = bits.sum(1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int().repeat(G * K, 1).to(DEV)
    got = ops.beam_candidates(rows, scores.to(DEV), candidates=n, allow_mask=words)
    want = ranked(x, allowed, G, K, n)
    assert [list(zip(b, t)) for b, t in zip(got.beams.tolist(), got.tokens.tolist())] == want


def test_a_step_of_equal_rows():
    G, K, V = 2, 32, 5000
    state = beam_start(G, K, DEV, all_beams=True)
    got = beam_step(torch.zeros(1, 1, V, dtype=BF, device=DEV).expand(G, K, V), state,
                    eos_token_id=1, pad_token_id=0)
    # beam 0's tokens, without its ending one; its best child keeps its slot
    for g in range(G):
        assert got.tokens.view(G, K)[g].tolist() == [0, *range(2, K + 1)]
    assert got.parents.view(G, K).eq(torch.arange(G, device=DEV).int().unsqueeze(1) * K).all()
    assert got.state.pool_steps[:, 0].eq(0).all() and got.state.pool_steps[:, 1:].eq(-1).all()


def test_references_that_lead_nowhere():
    """A pool entry of another group's row, or of a step that was not taken, has
    no tokens; a beam whose parents leave the group has padding ahead."""
    G, K, T, pad = 2, 3, 4, 77
    st = beam_start(G, K, DEV, all_beams=True)
    pool = torch.tensor([[-1.0, -2.0, -3.0]] * G, device=DEV)
    tokens = torch.full((T, G * K), 9, dtype=torch.int64, device=DEV)
    same = torch.arange(G * K, dtype=torch.int32, device=DEV).repeat(T, 1)
    rows = torch.tensor([[3, -1, 1 << 30], [2, 6, -(1 << 30)]], dtype=torch.int32, device=DEV)
    ok = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    step = torch.full((G, K), 2, dtype=torch.int32, device=DEV)
    for r, s in ((rows, step), (ok, step + 7), (ok, step - 9)):
        bad = st._replace(pool_scores=pool, pool_rows=r, pool_steps=s,
                          done=torch.ones_like(st.done), step=T)
        out = beam_finish(bad, tokens, same, eos_token_id=1, pad_token_id=pad, num_return=K)
        assert torch.equal(out.scores, pool)
        assert not out.lengths.any() and out.tokens.eq(pad).all()
    live = st._replace(scores=pool, step=T)
    out = beam_finish(live, tokens, torch.full_like(same, -5), eos_token_id=1, pad_token_id=pad,
                      num_return=K)
    assert out.tokens[..., :-1].eq(pad).all() and out.tokens[..., -1].eq(9).all()
