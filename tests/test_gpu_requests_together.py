"""The operators of a rollout of many requests run together: each request's
adapter beside the shared projection, its beams through one selection, its
states behind them; and the adapters of a training step from their forward to
the clipping.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd import decode_loop as dl
from graspo_amd import ops
from graspo_amd.beam_search import beam_start, beam_step, expand_states, reorder_states_
from graspo_amd.embedding import token_embedding
from graspo_amd.grad_clip import clip_grad_norm_
from graspo_amd.lora import lora_add
from graspo_amd.sft_loss import sft_cross_entropy_loss_from_hidden

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16
V, H, R, E, EOS, PAD = 503, 64, 8, 3, 5, 0


class AdapterLM:
    """A recurrent toy: state = tanh(state + rows), logits by a projection with
    each request's adapter; rows of a request follow one another."""

    def __init__(self, seed, ids):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.table = (rnd(V, H)).to(BF).to(DEV)
        self.head = (rnd(V, H) * 0.5).to(BF).to(DEV)
        self.a = (rnd(E, R, H) / H ** 0.5).to(BF).to(DEV)
        self.b = (rnd(E, V, R) * 0.7).to(BF).to(DEV)
        self.ids = ids.to(DEV)

    def __call__(self, tokens, attention_mask=None, past_key_values=None, use_cache=False):
        rows = tokens.shape[0]
        state = torch.zeros(rows, H, device=DEV) if past_key_values is None else past_key_values[0]
        x = token_embedding(tokens, self.table, check_status=False).float()
        live = attention_mask[:, -tokens.shape[1]:].unsqueeze(-1)
        for i in range(tokens.shape[1]):
            state = torch.where(live[:, i], torch.tanh(0.5 * state + x[:, i]), state)
        hidden = state.to(BF)
        base = torch.nn.functional.linear(hidden, self.head)
        ids = self.ids.repeat_interleave(rows // len(self.ids))
        logits = lora_add(base, hidden, self.a, self.b, adapter_ids=ids, scaling=0.5,
                          check_status=False)
        return logits.unsqueeze(1), (state,)


class Adapter:
    def __init__(self, model):
        self.model = model

    def _sync_timing(self):
        pass


def test_requests_beside_each_other_and_alone():
    ids = torch.tensor([0, 2, -1, 1, 2])
    g = torch.Generator().manual_seed(0)
    prompts = torch.randint(8, V, (5, 4), generator=g)
    args = dict(eos_token_id=EOS, pad_token_id=PAD, max_new_tokens=12, num_beams=4, num_return=2)
    together, scores, _ = dl.generate_beams_with_kv_cache(
        Adapter(AdapterLM(1, ids)), sequences=prompts.to(DEV), **args)
    seen = set()
    for i in range(5):
        alone, s, _ = dl.generate_beams_with_kv_cache(
            Adapter(AdapterLM(1, ids[i:i + 1])), sequences=prompts[i:i + 1].to(DEV), **args)
        n = alone.shape[1]
        assert torch.equal(together[2 * i:2 * i + 2, :n], alone)
        assert together[2 * i:2 * i + 2, n:].eq(PAD).all()
        # 12 steps' logits, each off by a bf16 rounding of the projection's own
        # sums in another order: 2^-8 of logits below 32
        assert (scores[i] - s[0]).abs().max() <= 2.0 ** -8 * 32
        seen.add(tuple(alone[0].tolist()[4:]))
    assert len(seen) > 1  # (the adapters do make a difference)


def test_a_step_captured_and_replayed():
    """Adapters, selection and states of one decode step in a graph, against
    the same calls outside of it."""
    G, K = 3, 4
    lm = AdapterLM(2, torch.tensor([1, 0, -1]))
    g = torch.Generator().manual_seed(3)
    rows = G * K
    hidden = (torch.randn(rows, H, generator=g)).to(BF).to(DEV)
    cache = [torch.randn(rows, 2, 9, 16, generator=g).to(BF).to(DEV) for _ in range(3)]
    ids = lm.ids.repeat_interleave(K)
    first = beam_start(G, K, DEV, all_beams=True)
    first = first._replace(scores=-torch.rand(G, K, generator=g).to(DEV))
    live = [t.clone() for t in first[:5]]

    def step(caches):
        base = torch.nn.functional.linear(hidden, lm.head)
        logits = lora_add(base, hidden, lm.a, lm.b, adapter_ids=ids, scaling=0.5)
        got = beam_step(logits, first._replace(scores=live[0], pool_scores=live[1],
                                               pool_rows=live[2], pool_steps=live[3],
                                               done=live[4]),
                        eos_token_id=EOS, pad_token_id=PAD)
        reorder_states_(caches, got.parents, K, check_status=False)
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in cache])
    torch.cuda.current_stream().wait_stream(side)
    moved = [t.clone() for t in cache]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(moved)
    for i in range(4):
        hidden.copy_(torch.randn(rows, H, generator=g).to(BF))
        live[0].copy_(-torch.rand(G, K, generator=g))
        for t, c in zip(moved, cache):
            t.copy_(c)
        want_cache = [t.clone() for t in cache]
        want = step(want_cache)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((got.tokens, got.parents, got.status, *got.state[:5]),
                        (want.tokens, want.parents, want.status, *want.state[:5])):
            assert torch.equal(a, b), i
        for a, b, c in zip(moved, want_cache, cache):
            assert torch.equal(a, b) and torch.equal(a, c[want.parents.long()])


def test_expanded_states_follow_like_the_originals():
    g = torch.Generator().manual_seed(4)
    prompt = [torch.randn(3, 2, 7, 8, generator=g).to(DEV) for _ in range(4)]
    states = expand_states(prompt, 5)
    parents = (torch.randint(0, 5, (3, 5), generator=g) + torch.arange(3)[:, None] * 5).flatten()
    reorder_states_(states, parents.to(DEV), 5)  # (the beams of a prompt are alike)
    for s, p in zip(states, prompt):
        assert torch.equal(s, p.repeat_interleave(5, 0))


@pytest.mark.parametrize("dtype", [BF, torch.float16], ids=["bf16", "fp16"])
def test_training_step_of_the_adapters(dtype):
    """Embedding, projection with adapters, mean loss from hidden states, the
    adapters' gradients, the global norm, the clipping: what autograd gives is
    what the operators give one after another, to the bit, and the norm is the
    gradients' within fp32 rounding."""
    g = torch.Generator().manual_seed(5)
    B, S = 3, 37
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    table, head = (rnd(V, H)).to(dtype).to(DEV), (rnd(V, 72) * 0.3).to(dtype).to(DEV)
    w = (rnd(72, H) / H ** 0.5).to(dtype).to(DEV)
    a = torch.nn.Parameter((rnd(E, R, H) / H ** 0.5).to(dtype).to(DEV))
    b = torch.nn.Parameter((rnd(E, 72, R) * 0.2).to(dtype).to(DEV))
    ids = torch.tensor([2, 0, 2]).to(DEV)
    scaling = torch.tensor([0.5, 1.0, 2.0], device=DEV)
    tokens = torch.randint(0, V, (B, S), generator=g).to(DEV)
    labels = tokens.clone()
    labels[:, :5] = -100

    x = token_embedding(tokens, table)
    base = torch.nn.functional.linear(x, w)
    hidden = lora_add(base, x, a, b, adapter_ids=ids, scaling=scaling)
    hidden.retain_grad()
    loss = sft_cross_entropy_loss_from_hidden(hidden, head, labels)
    loss.backward()

    with torch.no_grad():
        out, state = ops.lora_add_state(base, x, a, b, adapter_ids=ids, scales=scaling)
        gx, ga, gb = ops.lora_backward(hidden.grad, x, a, b, state, requests=3, need_x=False)
    assert torch.equal(out, hidden) and gx is None
    assert torch.equal(ga, a.grad) and torch.equal(gb, b.grad)
    assert not a.grad[1].any() and not b.grad[1].any()  # no row has adapter 1
    exact = float(sum(p.grad.double().square().sum() for p in (a, b)).sqrt())
    before = [p.grad.clone() for p in (a, b)]
    norm = clip_grad_norm_([a, b], exact / 3)
    assert abs(float(norm) - exact) <= exact * 2.0 ** -23
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for p, old in zip((a, b), before):
        # one fp32 factor, one product, one rounding
        want = old.double() * min(1.0, exact / 3 / (exact + 1e-6))
        assert ((p.grad.double() - want).abs() <= want.abs() * (u + 2.0 ** -21) + tiny).all()
