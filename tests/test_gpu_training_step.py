"""The operators around one tied vocabulary matrix run together, as a training
step runs them: the tokens looked up, token logprobs from the hidden states,
both gradients, the matrix's two gradients joined, the global norm clipped.

Tolerances: those of the logprobs from hidden states carried through the
lookup's gradient.  An element of it is s sum(gh): the hidden gradient's own
error summed, c w sum|gh| for c tokens in fp32, and one rounding, u; joining
it with the matrix product's rounds once more, u of the sum.
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.embedding import token_embedding
from graspo_amd.grad_clip import clip_grad_norm_
from graspo_amd.graspo_loss import sequence_log_probs_from_hidden
from graspo_amd.sft_loss import sft_cross_entropy_loss_from_hidden
from test_gpu_linear_logprob import W, expect, half_step, within

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
SCALE, PAD = 8.0, 0


def batch(B, S, V, H, dtype, seed):
    """(ids with right padding, table, gradient per predicted token)."""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, H, generator=g) / H ** 0.5).to(dtype)
    ids = torch.randint(1, V, (B, S), generator=g)
    grad = torch.randn(B, S - 1, generator=g) / (B * S)
    for b in range(1, B):
        n = int(torch.randint(2, S, (1,), generator=g))
        ids[b, n:] = PAD
        grad[b, n - 1:] = 0.0
    return ids, w, grad


def policy(ids, w):
    """The logprob of each next token; the hidden states are the rows."""
    rows = token_embedding(ids, w, scale=SCALE, padding_idx=PAD)
    return rows, sequence_log_probs_from_hidden(rows[:, :-1], w, ids[:, 1:])


def expect_step(ids, w, grad, dtype):
    """Logprobs and the tied gradient's two parts, with bounds, in 64 bits."""
    B, S = ids.shape
    V, H = w.shape
    u = half_step(dtype)
    rows = (w[ids].float() * SCALE).to(dtype)  # one product rounded once: exact to the bit
    lp, lp_e, gh, gh_e, gw, gw_e = expect(rows[:, :-1].reshape(-1, H), w, ids[:, 1:].reshape(-1),
                                          grad.reshape(-1), dtype)
    live = (ids[:, :-1] != PAD).reshape(-1)
    at = ids[:, :-1].reshape(-1)[live]
    total = lambda x: torch.zeros(V, H, dtype=torch.float64).index_add_(0, at, x[live]) * SCALE  # noqa: E731
    ge, mag, err = total(gh), total(gh.abs() + gh_e), total(gh_e)
    err = err + S * B * W * mag
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    ge_e = err + (u + 2 * W) * (ge.abs() + err) + tiny
    return rows, lp, lp_e, gw, gw_e, ge, ge_e


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,S,V,H", [(1, 2, 3, 8), (2, 9, 40, 64), (3, 50, 333, 72), (2, 200, 1000, 200)])
def test_tied_step(B, S, V, H, dtype):
    ids, w, grad = batch(B, S, V, H, dtype, seed=S + V)
    rows, lp, lp_e, gw, gw_e, ge, ge_e = expect_step(ids, w, grad, dtype)
    p = torch.nn.Parameter(w.cuda())
    got_rows, got = policy(ids.cuda(), p)
    assert torch.equal(got_rows.detach().cpu(), rows)
    within(got.detach().cpu().reshape(-1), lp, lp_e, "logprobs")
    (got * grad.cuda()).sum().backward()
    u, want = half_step(dtype), gw + ge
    err = gw_e + ge_e
    within(p.grad.cpu(), want, err + u * (want.abs() + err), "tied gradient")
    before = p.grad.clone()
    exact = float(before.double().square().sum().sqrt())
    norm = clip_grad_norm_([p], 0.5 * exact)
    assert abs(float(norm) - exact) <= 2 * W * exact
    # the factor is exact / 2 up to 1e-6 and three fp32 roundings
    f = 0.5 * exact / (exact + 1e-6)
    b = before.double()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    within(p.grad.cpu(), (b * f).cpu(), ((u + 6 * W) * b.abs() * f + tiny).cpu(), "clipped")


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_the_lookups_gradient_added_in_place(dtype):
    """Without a second [V, H] for it: onto the matrix product's, rounded once."""
    B, S, V, H = 2, 70, 400, 88
    ids, w, grad = batch(B, S, V, H, dtype, seed=4)
    rows, lp, lp_e, gw, gw_e, ge, ge_e = expect_step(ids, w, grad, dtype)
    d, wd = ids.cuda(), w.cuda().requires_grad_()
    out, bad, order = ops.embedding_ordered(d, wd.detach(), scale=SCALE, padding_idx=PAD)
    assert not bad
    hidden = out.requires_grad_()
    got = sequence_log_probs_from_hidden(hidden[:, :-1], wd, d[:, 1:])
    gh, g = torch.autograd.grad(got, [hidden, wd], grad.cuda())
    assert bool((gh[:, -1] == 0).all())
    ops.embedding_backward(None, gh, V, scale=SCALE, order=order, out=g)
    within(g.cpu(), gw + ge, gw_e + ge_e + 2 * W * gw.abs(), "tied gradient")


def test_steps_on_another_stream_repeat_to_the_bit():
    """Two passes of three optimizer steps, one of them on a side stream."""
    B, S, V, H = 4, 100, 2000, 128
    ids, w, _ = batch(B, S, V, H, BF, seed=6)
    labels = torch.where(ids == PAD, -100, ids).cuda()
    ids = ids.cuda()

    def steps():
        p, a = torch.nn.Parameter(w.cuda()), torch.nn.Parameter(torch.ones(H, device="cuda"))
        seen = []
        for _ in range(3):
            rows = token_embedding(ids, p, scale=SCALE, padding_idx=PAD)
            loss = sft_cross_entropy_loss_from_hidden((rows.float() * a).to(BF), p, labels)
            loss.backward()
            seen += [loss.detach(), clip_grad_norm_([p, a], 0.25)]
            with torch.no_grad():
                for x in (p, a):
                    x -= 0.1 * x.grad.to(x.dtype)
                    x.grad = None
        return [p.detach(), a.detach(), *seen]

    here = steps()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = steps()
    torch.cuda.synchronize()
    for x, y in zip(here, there):
        assert torch.equal(x, y) and bool(x.isfinite().all())


def test_steps_of_two_streams_at_once():
    """Neither waits for the other, and both get what they get alone."""
    sizes = [(2, 80, 3000, 256), (1, 200, 1500, 384)]
    made = []
    for i, (B, S, V, H) in enumerate(sizes):
        ids, w, grad = batch(B, S, V, H, BF, seed=60 + i)
        made.append((ids.cuda(), w.cuda().requires_grad_(), grad.cuda()))

    def step(ids, w, grad):
        _, lp = policy(ids, w)
        (g,) = torch.autograd.grad(lp, [w], grad)
        p = torch.nn.Parameter(w.detach(), requires_grad=False)
        p.grad = g
        return lp.detach(), clip_grad_norm_([p], 1e-3), g

    want = [[x.clone() for x in step(*m)] for m in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for m, s in zip(made, streams):
            with torch.cuda.stream(s):
                got.append(step(*m))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for x, y in zip(out, want[i % 2]):
            assert torch.equal(x, y)


def test_step_captured_and_replayed():
    B, S, V, H = 2, 60, 700, 64
    ids = torch.zeros(B, S, dtype=torch.int64, device="cuda")
    w = torch.zeros(V, H, dtype=BF, device="cuda").requires_grad_()
    grad = torch.zeros(B, S - 1, device="cuda")

    def fill(k):
        i, x, g = batch(B, S, V, H, BF, seed=30 + k)
        ids.copy_(i), grad.copy_(g)
        with torch.no_grad():
            w.copy_(x)

    def step():
        _, lp = policy(ids, w)
        (g,) = torch.autograd.grad(lp, [w], grad)
        p = torch.nn.Parameter(w.detach(), requires_grad=False)
        p.grad = g
        return lp.detach(), g, clip_grad_norm_([p], 1e-3)

    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for k in range(4):
        fill(k)
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        for graph, held in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(held, want):
                assert torch.equal(a, b)


def test_captures_beside_an_eager_graph_are_refused():
    ids = torch.arange(8, device="cuda").view(2, 4)
    w = torch.randn(20, 16, device="cuda").to(BF).requires_grad_()
    calls = [lambda: token_embedding(ids, w), lambda: sequence_log_probs_from_hidden(hidden, w, ids)]
    hidden = torch.randn(2, 4, 16, device="cuda").to(BF)
    for call in calls:
        eager = call()
        seen = []
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = hidden * 1.0  # (a graph is not captured empty)
            try:
                call()
            except RuntimeError as e:
                seen.append(str(e))
        assert len(seen) == 1 and "eager graph" in seen[0]
        del eager
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # one that a capture may join
            beside = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
            (g,) = torch.autograd.grad(out, [w], torch.ones_like(out))
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        want_out = call()
        (want,) = torch.autograd.grad(want_out, [w], torch.ones_like(want_out))
        assert torch.equal(out.detach(), want_out.detach()) and torch.equal(g, want)
        del out, want_out, kept, beside


def test_second_derivatives_are_refused():
    w = torch.randn(20, 8, device="cuda").requires_grad_()
    scale = torch.ones((), device="cuda", requires_grad=True)
    rows = token_embedding(torch.arange(5, device="cuda"), w)
    (g,) = torch.autograd.grad((rows * scale).sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    h = torch.randn(1, 4, 8, device="cuda").to(BF).requires_grad_()
    lp = sequence_log_probs_from_hidden(h, w.detach().to(BF), torch.arange(4, device="cuda").view(1, 4))
    (g,) = torch.autograd.grad((lp * scale).sum(), [h], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
