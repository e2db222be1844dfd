"""A beam search's step against its definition in 64 bits.

Scores: c = score + x - lse, lse from a sum of fp32 exponentials.  Each is off
by one part in 2^23 (the exponential) and 0.7 |arg| in 2^24 (its argument's
rounding, |arg| < 64 where it matters), a lane adds at most 8 + V / 2048 of
them and a few partial sums, half a step each: below 256 * 2^-24 in all for
V <= 2^18, and c itself is rounded once.  Two candidates whose exact scores
are further apart than twice that have to come in their order.
"""

from __future__ import annotations

import io
import math

import pytest
import torch

from graspo_amd import ops
from graspo_amd.beam_search import (BeamState, beam_finish, beam_start, beam_step, length_of)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
INF = math.inf
BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32


def tol(c):
    return 256 * 2.0 ** -24 + abs(c) * 2.0 ** -24 if math.isfinite(c) else 0.0


def pack(allowed):
    """bool [R, V] -> int32 [R, ceil(V / 32)]"""
    R, V = allowed.shape
    w = torch.nn.functional.pad(allowed, (0, -V % 32)).view(R, -1, 32).long()
    w = (w << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def exact(x, scores, allowed=None, done=None):
    """c [G, K * V] in 64 bits; -inf where there is no candidate."""
    G, K = scores.shape
    x = x.double().reshape(G, K, -1)
    bad = ~(x < INF).all(-1, keepdim=True)
    c = scores.double().unsqueeze(-1) + torch.log_softmax(x, -1)
    if allowed is not None:
        c = c.masked_fill(~allowed.view(c.shape), -INF)
    c = c.masked_fill(bad | ~scores.isfinite().unsqueeze(-1) | c.isnan(), -INF)
    if done is not None:
        c = c.masked_fill(done.view(-1, 1, 1), -INF)
    return c.reshape(G, -1)


def check(x, scores, n=None, allowed=None, done=None, given=None):
    G, K = scores.shape
    V = x.shape[-1]
    n = 2 * K if n is None else n
    got = ops.beam_candidates(given if given is not None else x.to(DEV), scores.to(DEV),
                              candidates=n,
                              allow_mask=None if allowed is None else pack(allowed).to(DEV),
                              done=None if done is None else done.to(DEV))
    s, b, t = (v.cpu() for v in got[:3])
    assert s.shape == b.shape == t.shape == (G, n)
    for g, c in enumerate(exact(x, scores, allowed, done)):
        want, at = torch.sort(c, descending=True, stable=True)
        want, at = want[:n + 1].tolist(), at[:n + 1].tolist()
        want += [-INF] * (n + 1 - len(want))
        seen = set()
        for i in range(n):
            if want[i] == -INF:
                assert (float(s[g, i]), int(b[g, i]), int(t[g, i])) == (-INF, -1, -1), (g, i)
                continue
            flat = int(b[g, i]) * V + int(t[g, i])
            assert 0 <= int(b[g, i]) < K and 0 <= int(t[g, i]) < V and flat not in seen
            seen.add(flat)
            e = tol(want[i])
            assert abs(float(s[g, i]) - want[i]) <= e, (g, i, float(s[g, i]), want[i])
            assert abs(float(c[flat]) - want[i]) <= 2 * e, (g, i)
            # an order that the rounding cannot change, and ties of one row
            near = [j for j in range(n + 1) if j != i and want[j] > -INF
                    and abs(want[j] - want[i]) <= 2 * e
                    and not (want[j] == want[i] and at[j] // V == at[i] // V)]
            if not near:
                assert flat == at[i], (g, i, flat, at[i])
    return got


def rows(G, K, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(G * K, V, generator=g) * 3).to(dtype)
    scores = -torch.rand(G, K, generator=g) * 20
    return x, scores


@pytest.mark.parametrize("dtype", [BF, HF, F4], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("G,K,V", [
    (1, 1, 1), (1, 2, 3), (3, 2, 5), (2, 4, 64), (1, 3, 511), (2, 5, 513), (3, 4, 2048),
    (1, 8, 4099), (2, 16, 8191), (1, 32, 20001), (5, 3, 50257), (1, 4, 151936), (9, 2, 32000),
])
def test_candidates(G, K, V, dtype):
    print("candidates", G, K, V, dtype, flush=True)
    x, scores = rows(G, K, V, dtype, seed=V + K)
    got = check(x, scores)
    assert not got.status.any()


@pytest.mark.parametrize("n", [1, 2, 7, 33, 64])
def test_numbers_of_candidates(n):
    for G, K, V in [(2, 3, 9), (2, 1, 5000), (1, 32, 3000)]:
        x, scores = rows(G, K, V, BF, seed=n)
        check(x, scores, n=n)


def test_a_large_batch():
    x, scores = rows(32, 8, 40000, BF, seed=5)
    check(x, scores)


@pytest.mark.parametrize("dtype", [BF, F4], ids=["bf16", "fp32"])
def test_equal_logits_go_by_beam_and_token(dtype):
    print("ties", dtype, flush=True)
    # all alike; two values; rising and falling rows (each lane's last is its best)
    V = 9000
    for x in (torch.zeros(1, V), torch.full((1, V), -0.0), (torch.arange(V) % 2).float()[None],
              torch.arange(V).float()[None] / 64, -torch.arange(V).float()[None] / 64,
              torch.full((1, V), 3.0).index_fill_(1, torch.tensor([4097]), -0.0)):
        x = x.to(dtype).repeat(4, 1)
        for scores in (torch.zeros(1, 4), torch.tensor([[-1.0, 0.0, -1.0, 0.0]])):
            s, b, t, _ = ops.beam_candidates(x.to(DEV), scores.to(DEV))
            # equal rows have equal sums to the bit: beams tie exactly
            c = exact(x, scores)[0]
            at = torch.sort(c, descending=True, stable=True).indices[:8]
            assert (b[0].cpu().long() * V + t[0].cpu()).tolist() == at.tolist()
    # zeros of both signs are equal
    x = torch.full((1, V), -0.0)
    x[0, 5000:] = 0.0
    t = ops.beam_candidates(x.to(dtype).to(DEV), torch.zeros(1, 1, device=DEV), candidates=5)[2]
    assert t.tolist() == [[0, 1, 2, 3, 4]]


@pytest.mark.parametrize("dtype", [BF, HF, F4], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("share", [0.0, 0.0005, 0.02, 0.5, 1.0])
def test_masks(share, dtype):
    print("mask", share, dtype, flush=True)
    for G, K, V in [(2, 3, 7), (2, 4, 5003), (1, 2, 70000)]:
        x, scores = rows(G, K, V, dtype, seed=17)
        g = torch.Generator().manual_seed(int(share * 1e4))
        allowed = torch.rand(G * K, V, generator=g) < share
        allowed[0] = False  # a row that the mask leaves nothing
        got = check(x, scores, allowed=allowed)
        want = torch.where(allowed.any(1), ops.ROW_OK, ops.ROW_EMPTY)
        assert torch.equal(got.status.cpu().long(), want)


def test_masked_values_of_every_kind():
    # the lowest value, -inf and huge values under the mask and beside it
    x, scores = rows(1, 4, 6000, BF, seed=3)
    x[0, :3000] = -INF
    x[1, ::2] = torch.finfo(BF).min
    x[2, 5] = 1e30  # takes all of the softmax
    x[3] = -INF
    x[3, 4567] = -2.0
    got = check(x, scores)
    assert not got.status.any()
    allowed = torch.ones(4, 6000, dtype=torch.bool)
    allowed[2, 5] = False
    allowed[3, 4567] = False
    got = check(x, scores, allowed=allowed)
    assert got.status.tolist() == [0, 0, 0, ops.ROW_EMPTY]


def test_rows_that_are_not_finite():
    x, scores = rows(2, 3, 4000, F4, seed=8)
    x[0, 17] = float("nan")
    x[1, 3999] = INF
    x[2] = -INF
    x[3] = float("nan")
    scores[1, 1] = -INF  # dead beams are not read
    x[4, 5] = float("nan")
    got = check(x, scores)
    nf = ops.ROW_NONFINITE
    assert got.status.tolist() == [nf, nf, ops.ROW_EMPTY, nf, 0, 0]
    scores[1, 2] = float("nan")
    scores[0, 0] = INF
    got = check(x, scores)
    assert got.status.tolist() == [nf, nf, ops.ROW_EMPTY, nf, 0, nf]
    assert got.beams.eq(-1).all()
    done = torch.tensor([False, True])
    assert check(x, scores, done=done).status.tolist() == [nf, nf, ops.ROW_EMPTY, 0, 0, 0]


def test_layouts():
    G, K, V = 3, 4, 1003
    for dtype in (BF, F4):
        for off in (0, 1, 3):
            buf = torch.zeros(G * K * (V + 17) * 2 + 8, dtype=dtype, device=DEV)
            x, scores = rows(G, K, V, dtype, seed=off)
            # rows apart, groups apart, at any element
            v = buf[off:off + G * K * (V + 17)].view(G * K, V + 17)[:, :V]
            v.copy_(x)
            check(x, scores, given=v)
            v = buf[off:off + G * K * (V + 17) * 2].view(G, 2, K, V + 17)[:, 1, :, :V]
            v.copy_(x.view(G, K, V))
            check(x, scores, given=v)
            # the prompt's row for all of its beams
            one = x[:G]
            scores[:, 1:] = -INF
            check(one.repeat_interleave(K, 0), scores,
                  given=one.to(DEV).unsqueeze(1).expand(G, K, V))


def test_steps_without_a_group():
    st = beam_start(0, 4, DEV)
    got = beam_step(torch.zeros(0, 50, device=DEV), st, eos_token_id=1, pad_token_id=0)
    assert got.tokens.shape == (0,) and got.state.scores.shape == (0, 4) and got.state.step == 1
    cand = ops.beam_candidates(torch.zeros(0, 50, device=DEV), st.scores)
    assert ops.beam_advance(cand, *st[:5], eos_token_id=1, pad_token_id=0, length=1.0,
                            step=0).done.shape == (0,)
    none = torch.zeros(1, 0, dtype=torch.int64, device=DEV)
    out = beam_finish(got.state, none, none.int(), eos_token_id=1, pad_token_id=0)
    assert out.tokens.shape == (0, 1, 1)


def test_no_groups_and_no_live_beam():
    out = ops.beam_candidates(torch.zeros(0, 50, device=DEV), torch.zeros(0, 4, device=DEV))
    assert out.scores.shape == (0, 8)
    dead = torch.full((2, 4), -INF, device=DEV)
    out = ops.beam_candidates(torch.zeros(8, 50, device=DEV), dead)
    assert out.beams.eq(-1).all() and not out.status.any()


def test_offsets_past_32_bits():
    # rows that begin past 2^32 bytes, and past 2^31 elements
    G, K, V = 1, 3, 5000
    x, scores = rows(G, K, V, BF, seed=1)
    buf = torch.zeros(K, (1 << 30) + (1 << 29), dtype=BF, device=DEV)
    v = buf[:, :V]
    v.copy_(x)
    check(x, scores, given=v)


# ----------------------------------------------------------------- a step

def f32(v):
    return float(torch.tensor(v, dtype=torch.float64).float())


def advance(cand, scores, pool, done, eos, pad, length, step, early):
    """One group by the rules; cand: (score, beam, token), pool: (score, row in
    the group, step)."""
    K = len(scores)
    if done:
        return [pad] * K, list(range(K)), list(scores), pool, True
    live, pool = [], list(pool)
    for rank, (s, b, t) in enumerate(cand):
        if b >= 0 and t == eos:
            if rank < K:
                pool.append((f32(s / length), b, step))
        elif len(live) < K:
            live.append((s, b, t))
    pool = [h for h in sorted(pool, key=lambda h: -h[0])[:K] if h[0] > -INF]
    slot, rest = {}, []
    for c in live:
        if c[1] >= 0 and c[1] not in slot:
            slot[c[1]] = c
        else:
            rest.append(c)
    for k in range(K):
        if k not in slot:
            c = rest.pop(0) if rest else (-INF, -1, -1)
            slot[k] = c if c[1] >= 0 else (-INF, k, pad)
    out = [slot[k] for k in range(K)]
    best = max(s for s, _, _ in out)
    full = len(pool) == K and (early or pool[-1][0] >= f32(best / length))
    return [t for _, _, t in out], [b for _, b, _ in out], [s for s, _, _ in out], pool, \
        full or best == -INF


def state_of(G, K, seed, step, dead=0.0):
    g = torch.Generator().manual_seed(seed)
    scores = -torch.rand(G, K, generator=g) * 5
    scores[torch.rand(G, K, generator=g) < dead] = -INF
    filled = torch.randint(0, K + 1, (G, 1), generator=g)
    has = torch.arange(K)[None] < filled
    pool = (-torch.rand(G, K, generator=g) * 2).sort(dim=1, descending=True).values
    rows_ = torch.randint(0, K, (G, K), generator=g) + torch.arange(G)[:, None] * K
    steps = torch.randint(0, max(step, 1), (G, K), generator=g)
    return BeamState(scores, torch.where(has, pool, -INF), torch.where(has, rows_, -1).int(),
                     torch.where(has, steps, -1).int(), torch.rand(G, generator=g) < 0.15, step)


def on(state, dev):
    return BeamState(*(v.to(dev) for v in state[:5]), state.step)


def check_step(x, st, eos, pad, penalty, early, allowed=None):
    G, K = st.scores.shape
    mask = None if allowed is None else pack(allowed).to(DEV)
    dev = on(st, DEV)
    got = beam_step(x.to(DEV), dev, eos_token_id=eos, pad_token_id=pad, length_penalty=penalty,
                    early_stopping=early, allow_mask=mask)
    cand = ops.beam_candidates(x.to(DEV), dev.scores, allow_mask=mask, done=dev.done)
    length = length_of(st.step + 1, penalty)
    two = ops.beam_advance(cand, *dev[:5], eos_token_id=eos, pad_token_id=pad, length=length,
                           step=st.step, early_stopping=early)
    for a, b in zip((got.tokens, got.parents, *got.state[:5]), two):
        assert torch.equal(a, b)
    assert torch.equal(got.status, cand.status) and got.state.step == st.step + 1
    c = [v.cpu().tolist() for v in cand[:3]]
    for g in range(G):
        pool = [(s, r - g * K, t) for s, r, t in zip(*(v[g].tolist() for v in st[1:4])) if s > -INF]
        want = advance(list(zip(c[0][g], c[1][g], c[2][g])), st.scores[g].tolist(), pool,
                       bool(st.done[g]), eos, pad, length, st.step, early)
        assert got.tokens.view(G, K)[g].tolist() == want[0]
        assert (got.parents.view(G, K)[g] - g * K).tolist() == want[1]
        assert got.state.scores[g].tolist() == want[2]
        empty = [(-INF, -1 - g * K, -1)] * (K - len(want[3]))
        rows_ = (got.state.pool_rows[g].cpu() - g * K).tolist()
        have = list(zip(got.state.pool_scores[g].tolist(), rows_, got.state.pool_steps[g].tolist()))
        assert have == want[3] + empty
        assert bool(got.state.done[g]) == want[4]
    p = got.parents.long()
    assert torch.equal(p[p], p)
    return got


@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("G,K,V", [(1, 1, 40), (7, 2, 30), (6, 3, 9), (9, 4, 777), (5, 8, 300),
                                   (3, 16, 64), (2, 32, 5000), (4, 5, 3), (3, 4, 1)])
def test_step(G, K, V, early):
    print("step", G, K, V, early, flush=True)
    for i, (dead, bias, penalty) in enumerate([(0.0, 0.0, 1.0), (0.3, 4.0, 0.0), (0.0, 6.0, 0.6),
                                               (1.0, 0.0, 1.0), (0.7, 5.0, -1.0)]):
        x, _ = rows(G, K, V, BF, seed=i)
        eos = V // 2
        x[:, eos] += bias
        check_step(x, state_of(G, K, i, 3 * i, dead), eos, 1, penalty, early)


def test_step_with_masks():
    for share in (0.0, 0.002, 0.05):
        x, _ = rows(4, 3, 999, HF, seed=2)
        allowed = torch.rand(12, 999, generator=torch.Generator().manual_seed(2)) < share
        allowed[:, 0] |= torch.arange(12) % 2 == 0
        check_step(x, state_of(4, 3, 1, 5), 0, 7, 1.0, False, allowed)


def test_first_step_has_one_live_beam():
    st = beam_start(3, 4, "cpu")
    x, _ = rows(3, 4, 100, BF, seed=0)
    got = check_step(x, st, 99, 0, 1.0, False)
    assert got.parents.view(3, 4).eq(torch.arange(3, device=DEV).view(3, 1) * 4).all()


def test_no_candidate_at_all_is_done():
    st = beam_start(2, 3, "cpu")
    x = torch.full((6, 50), -INF)
    got = check_step(x, st, 9, 0, 1.0, False)
    assert got.state.done.all() and got.tokens.eq(0).all()
    assert got.status.tolist() == [ops.ROW_EMPTY, 0, 0] * 2


def test_the_same_bits_every_time():
    x, scores = rows(4, 4, 100000, BF, seed=9)
    x, scores = x.to(DEV), scores.to(DEV)
    first = ops.beam_candidates(x, scores)
    # whichever rows are beside it
    alone = ops.beam_candidates(x[:4], scores[:1])
    for _ in range(3):
        for a, b in zip(first, ops.beam_candidates(x, scores)):
            assert torch.equal(a, b)
    assert torch.equal(first.tokens[:1], alone.tokens)


def test_captured_and_replayed():
    G, K, V = 2, 4, 40000
    x, _ = rows(G, K, V, BF, seed=4)
    xd = x.to(DEV)
    st = on(state_of(G, K, 4, 2), DEV)
    args = dict(eos_token_id=5, pad_token_id=0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beam_step(xd, st, **args)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of the same call
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = beam_step(xd, st, **args)
        graphs.append((graph, out))
    for i in range(4):
        xd.copy_(rows(G, K, V, BF, seed=i)[0])
        want = beam_step(xd, st, **args)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip((out.tokens, out.parents, *out.state[:5]),
                            (want.tokens, want.parents, *want.state[:5])):
                assert torch.equal(a, b), i


def test_another_stream():
    x, scores = rows(2, 4, 60000, BF, seed=6)
    want = ops.beam_candidates(x.to(DEV), scores.to(DEV))
    side = torch.cuda.Stream()
    xs = torch.empty_like(x, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        xs.copy_(x.to(DEV, non_blocking=True))
        got = ops.beam_candidates(xs, scores.to(DEV))
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------- finish

def finish(st, tokens, parents, eos, pad, length, give):
    G, K = st.scores.shape
    T = st.step
    outs = []
    for g in range(G):
        hyps = [(s, r, t) for s, r, t in zip(*(v[g].tolist() for v in st[1:4])) if s > -INF]
        if not st.done[g] and T:
            hyps += [(f32(s / length), g * K + k, T)
                     for k, s in enumerate(st.scores[g].tolist()) if s > -INF]
        hyps = sorted(hyps, key=lambda h: -h[0])[:give]
        for s, row, t in hyps + [(-INF, None, None)] * (give - len(hyps)):
            if row is None:
                outs.append((s, 0, [pad] * T))
                continue
            seq = [eos] if t < T else []
            for i in range(t - 1, -1, -1):
                seq.append(int(tokens[i, row]))
                row = int(parents[i, row])
            seq.reverse()
            outs.append((s, len(seq), seq + [pad] * (T - len(seq))))
    return outs


@pytest.mark.parametrize("G,K,T,give", [(1, 1, 1, 1), (2, 3, 0, 2), (3, 4, 7, 4), (2, 32, 50, 20),
                                        (5, 2, 300, 1)])
def test_finish(G, K, T, give):
    g = torch.Generator().manual_seed(T)
    st = state_of(G, K, T, T, dead=0.3)
    if T == 0:
        st = beam_start(G, K, "cpu")
    tokens = torch.randint(2, 99, (T, G * K), generator=g)
    parents = (torch.randint(0, K, (T, G, K), generator=g)
               + torch.arange(G)[:, None] * K).reshape(T, G * K).int()
    got = beam_finish(on(st, DEV), tokens.to(DEV), parents.to(DEV), eos_token_id=1, pad_token_id=0,
                      length_penalty=0.7, num_return=give)
    want = finish(st, tokens, parents, 1, 0, length_of(max(T, 1), 0.7), give)
    s, n, t = got.scores.flatten().tolist(), got.lengths.flatten().tolist(), got.tokens.flatten(0, 1)
    assert list(zip(s, n, t.tolist())) == want


def test_finish_of_references_out_of_range():
    # rows and parents that are not the group's give no tokens, and no fault
    st = on(state_of(2, 3, 1, 4), DEV)
    st = st._replace(pool_rows=torch.full_like(st.pool_rows, 1 << 30),
                     pool_steps=torch.full_like(st.pool_steps, 9), done=torch.zeros_like(st.done))
    tokens = torch.ones(4, 6, dtype=torch.int64, device=DEV)
    parents = torch.full((4, 6), -5, dtype=torch.int32, device=DEV)
    out = beam_finish(st, tokens, parents, eos_token_id=1, pad_token_id=0, num_return=3)
    assert out.tokens.ge(0).all()


def test_outputs_have_storages_of_their_own():
    G, K, V = 3, 4, 500
    x = torch.randn(G * K, V, device=DEV)
    got = beam_step(x, beam_start(G, K, DEV, all_beams=True), eos_token_id=1, pad_token_id=0)
    outs = [got.tokens, got.parents, *got.state[:5], got.status]
    assert len({t.untyped_storage().data_ptr() for t in outs}) == len(outs)
    for t in outs:
        assert t.storage_offset() == 0
        assert t.untyped_storage().nbytes() == t.numel() * t.element_size()
    f = io.BytesIO()
    torch.save(outs, f)
    f.seek(0)
    assert all(torch.equal(a, b) for a, b in zip(torch.load(f, weights_only=True), outs))
