"""The beam-search loop with everything that it calls, over a model whose cache
holds what it has read: the logits depend on the cached tokens, so beams whose
states were not moved with them would go elsewhere.  The search is restated on
the host from the same logits, in 64 bits; the scores are compared within
the steps' summed tolerances, the tokens exactly (the seeds have no near-ties).
"""

from __future__ import annotations

import math
from collections import namedtuple

import pytest
import torch

from graspo_amd import decode_loop as dl
from graspo_amd.beam_search import length_of

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
V, EOS, PAD = 211, 7, 0
Layer = namedtuple("Layer", "keys values")


class CacheLM:
    """Logits of a row: a table's line by a hash of all tokens that its cache
    holds under the attention mask."""

    def __init__(self, seed, eos_bias, nan_at=None):
        g = torch.Generator().manual_seed(seed)
        self.table = (torch.randn(997, V, generator=g) * 2.0).to(torch.bfloat16)
        self.table[:, EOS] += eos_bias
        self.dev = self.table.to(DEV)
        self.nan_at, self.calls = nan_at, 0

    @staticmethod
    def hash(tokens, mask):
        n = tokens.shape[1]
        w = (torch.arange(1, n + 1, device=tokens.device) * 37) % 991
        return (torch.where(mask, tokens + 1, 0) * w).sum(1) % 997

    def __call__(self, ids, attention_mask=None, past_key_values=None, use_cache=False):
        assert use_cache and bool(((ids >= 0) & (ids < V)).all())
        rows = ids.shape[0]
        new = ids.to(torch.float32).view(rows, 1, -1, 1).expand(rows, 2, -1, 8)
        if past_key_values is None:
            keys, total = new.contiguous(), ids.sum(1).to(torch.int64)
        else:
            layer, extra = past_key_values
            assert layer.values is None and extra["length"] == layer.keys.shape[2]
            keys = torch.cat([layer.keys, new], 2)
            total = extra["total"] + ids.sum(1)
        tokens = keys[:, 1, :, 3].to(torch.int64)
        assert attention_mask.shape == tokens.shape
        # the recurrent state and the keys went the same way
        assert torch.equal(total, tokens.sum(1))
        out = self.dev[self.hash(tokens, attention_mask)]
        if self.nan_at == self.calls:
            out = out.clone()
            out[0, 3] = float("nan")
        self.calls += 1
        return (out.unsqueeze(1).expand(-1, ids.shape[1], -1),
                (Layer(keys, None), {"total": total, "length": keys.shape[2]}))


class Adapter:
    def __init__(self, model):
        self.model = model

    def _sync_timing(self):
        pass


def search(lm, prompt, K, T, penalty, early, give):
    """One prompt's beam search on the host: hypotheses as lists of tokens."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float64).float())  # noqa: E731
    beams, pool = [(0.0, [])] + [(-math.inf, [])] * (K - 1), []
    live_mask = prompt.ne(PAD)
    steps = 0
    for t in range(T):
        steps = t + 1
        cand = []
        for k, (s, toks) in enumerate(beams):
            if s == -math.inf:
                continue
            full = torch.cat([prompt, torch.tensor(toks, dtype=torch.int64)])
            mask = torch.cat([live_mask, torch.ones(len(toks), dtype=torch.bool)])
            x = lm.table[CacheLM.hash(full[None], mask[None])[0]].double()
            lp = torch.log_softmax(x, 0) + s
            cand += [(float(c), k, v) for v, c in enumerate(lp.tolist())]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        gaps = [a[0] - b[0] for a, b in zip(cand[:2 * K], cand[1:2 * K + 1])]
        assert min(g for g in gaps if g > 0) > 2e-5 or min(gaps) == 0.0
        length = length_of(t + 1, penalty)
        live = []
        for rank, (s, k, v) in enumerate(cand[:2 * K]):
            if v == EOS:
                if rank < K:
                    pool.append((f32(f32(s) / length), beams[k][1] + [v]))
            elif len(live) < K:
                live.append((k, f32(s), beams[k][1] + [v]))
        pool = sorted(pool, key=lambda h: -h[0])[:K]
        slots, rest = {}, []
        for k, s, toks in live:
            if k in slots:
                rest.append((s, toks))
            else:
                slots[k] = (s, toks)
        beams = [slots[k] if k in slots else rest.pop(0) if rest else (-math.inf, [])
                 for k in range(K)]
        best = max(s for s, _ in beams)
        if len(pool) == K and (early or pool[-1][0] >= f32(best / length)):
            return sorted(pool, key=lambda h: -h[0])[:give], steps
    if steps:
        pool = pool + [(f32(s / length_of(steps, penalty)), t) for s, t in beams if s > -math.inf]
    return sorted(pool, key=lambda h: -h[0])[:give], steps


def prompts(G, S, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(8, V, (G, S), generator=g)
    for b in range(1, G):
        p[b, : (b * 2) % S] = PAD  # padded on the left
    return p


@pytest.mark.parametrize("G,K,T,bias,penalty,early,give", [
    (1, 1, 6, 0.0, 1.0, False, 1), (2, 3, 9, 3.0, 1.0, False, 2), (3, 4, 12, 5.0, 0.6, False, 4),
    (2, 4, 12, 6.0, 1.0, True, 1), (2, 8, 7, 2.0, 0.0, False, 3), (4, 2, 1, 4.0, 1.0, False, 2),
    (1, 16, 10, 7.0, 1.2, False, 16),
])
def test_search(G, K, T, bias, penalty, early, give):
    print("beam loop", G, K, T, flush=True)
    lm = CacheLM(G * 100 + K, bias)
    p = prompts(G, 5, seed=K)
    seq, scores, timings = dl.generate_beams_with_kv_cache(
        Adapter(lm), sequences=p.to(DEV), eos_token_id=EOS, pad_token_id=PAD, max_new_tokens=T,
        num_beams=K, num_return=give, length_penalty=penalty, early_stopping=early)
    want = [search(lm, p[g], K, T, penalty, early, give) for g in range(G)]
    assert timings["decode_tokens"] == max(n for _, n in want)
    assert scores.shape == (G, give) and seq.shape[0] == G * give and seq.dtype == torch.int64
    longest = max(len(t) for hyps, _ in want for _, t in hyps)
    assert seq.shape[1] == 5 + longest
    seq, scores = seq.cpu(), scores.cpu()
    for g, (hyps, _) in enumerate(want):
        assert len(hyps) == give
        for i, (s, toks) in enumerate(hyps):
            row = seq[g * give + i]
            assert row[:5].tolist() == p[g].tolist()
            assert row[5:].tolist() == toks + [PAD] * (longest - len(toks)), (g, i)
            # each step's score is off by 256 steps of 2^-24 and one rounding
            off = len(toks) * (256 + 40) * 2.0 ** -24 / length_of(len(toks), penalty) * 2
            assert abs(float(scores[g, i]) - s) <= off + abs(s) * 2.0 ** -22


def test_nothing_to_generate():
    lm = CacheLM(1, 0.0)
    p = prompts(2, 5, 1).to(DEV)
    seq, scores, timings = dl.generate_beams_with_kv_cache(
        Adapter(lm), sequences=p, eos_token_id=EOS, pad_token_id=PAD, max_new_tokens=0,
        num_beams=3)
    assert torch.equal(seq, p) and timings["decode_tokens"] == 0 and scores.shape == (2, 1)


def test_a_row_that_is_not_finite_raises():
    for at in (0, 3):
        with pytest.raises(RuntimeError, match="non-finite"):
            dl.generate_beams_with_kv_cache(
                Adapter(CacheLM(3, 0.0, nan_at=at)), sequences=prompts(2, 5, 1).to(DEV),
                eos_token_id=EOS, pad_token_id=PAD, max_new_tokens=8, num_beams=3)


def test_arguments():
    a = Adapter(CacheLM(1, 0.0))
    args = dict(sequences=prompts(2, 5, 1).to(DEV), eos_token_id=EOS, pad_token_id=PAD,
                max_new_tokens=4)
    for bad in (dict(num_beams=0), dict(num_beams=33, num_return=1), dict(num_beams=2, num_return=3),
                dict(num_beams=2, num_return=0), dict(num_beams=2, length_penalty=1e6)):
        with pytest.raises(ValueError):
            dl.generate_beams_with_kv_cache(a, **args, **bad)
