"""Token logprobs and losses from hidden states, without the logits, against
the formulas in 64 bits.

Tolerances, from u = finfo(type).eps / 2 (half a step of the operands' type)
and w = 2^-24 (fp32):

- a logit is a sum of K exact products in fp32, within K w sum|h||w| of exact;
  the exponentials' arguments and the logarithm add at most 4 w (1 + max|x|),
  the sums of at most V positive terms V w relative (never more than 2^-12
  here, pairwise far less: 64 w is used for the folds of 16, 4 and 2 and the
  merges);
- an element of the logits' gradient d = g ([v = t] - p) is rounded once to
  the operands' type: u |d|, plus g p times twice the logits' error, plus, for
  fp16, half its smallest step at the power of two in it;
- (up to 128 rows D is kept in two parts of the type, the second one rounded:
  u^2 |d|, test_few_rows_keep_d_whole);
- a gradient sums N or V such products in fp32 and is rounded once: n w
  sum|d||x| and u |result| (and half the smallest step of the type).
"""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.graspo_loss import sequence_log_probs_from_hidden
from graspo_amd.sft_loss import sft_cross_entropy_loss_from_hidden

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
BF, HF = torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(N, V, K, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, K, generator=g) * spread / K ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    h = (torch.randn(N, K, generator=g) + w[t].float() * torch.rand(N, 1, generator=g) * 3).to(dtype)
    grad = torch.randn(N, generator=g) * 10.0 ** (-3 * torch.rand(N, generator=g))
    grad[torch.rand(N, generator=g) < 0.2] = 0.0
    return h, w, t, grad


def expect(h, w, t, g, dtype, parts=1):
    """(logprob, its bound, dh, its bound, dw, its bound) in 64 bits; D in
    `parts` of the type."""
    u, K, V = half_step(dtype), h.shape[1], w.shape[0]
    h, w, g = h.double(), w.double(), g.double()
    x, mag = h @ w.T, h.abs() @ w.abs().T
    lse = torch.logsumexp(x, 1)
    x_err = K * W * mag.amax(1) + 4 * W * (1 + x.abs().amax(1))
    lp = x.gather(1, t[:, None]).squeeze(1) - lse
    lp_err = 2 * x_err + 64 * W + 2 * W * lp.abs()
    p = (x - lse[:, None]).exp()
    d = -g[:, None] * p
    d.scatter_add_(1, t[:, None], g[:, None])
    d_err = u ** parts * d.abs() + (1 + u) * g.abs()[:, None] * p * 2 * (x_err + 64 * W)[:, None]
    # (1 - p and the product are fp32 operations too)
    d_err += 2 * W * g.abs()[:, None] * (t[:, None] == torch.arange(V, device=t.device)[None, :])
    if dtype == HF:
        d_err += g.abs().max() * 2.0 ** (1 - 15) * 2.0 ** -25
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    out = [lp, lp_err]
    for a, e, b in ((d, d_err, w), (d.T, d_err.T, h)):
        r = a @ b
        n = a.shape[1]
        err = e @ b.abs() + n * W * ((a.abs() + e) @ b.abs())
        out += [r, err + u * (r.abs() + err) + tiny]
    return out


def within(got, want, err, what):
    bad = ~((got.double().to(want.device) - want).abs() <= err)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double().to(want.device) - want).abs() / err).max()))


SIZES = [
    # N, V, K
    (1, 1, 8), (1, 7, 64), (2, 256, 128), (61, 257, 72), (255, 300, 64), (256, 255, 192),
    (257, 1000, 136), (600, 513, 328), (3, 5000, 100), (33, 777, 1), (130, 1025, 130),
    (40, 600, 2816), (5, 50257, 264),
]


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N,V,K", SIZES)
def test_logprob_and_gradients(N, V, K, dtype):
    h, w, t, g = inputs(N, V, K, dtype, seed=N + V + K)
    lp, lp_e, gh, gh_e, gw, gw_e = expect(h, w, t, g, dtype)
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    got = sequence_log_probs_from_hidden(hd, wd, t.cuda())
    within(got.detach().cpu(), lp, lp_e, "logprob")
    a, b = torch.autograd.grad(got, [hd, wd], g.cuda())
    assert a.dtype == dtype and a.shape == h.shape and b.dtype == dtype and b.shape == w.shape
    within(a.cpu(), gh, gh_e, "hidden's gradient")
    within(b.cpu(), gw, gw_e, "weight's gradient")


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N,V,K", [
    (64, 129, 256), (65, 128, 64), (127, 1000, 30), (128, 513, 1032), (129, 300, 72), (100, 33, 7),
    (64, 1, 520), (16, 4097, 1),
])
def test_few_rows(N, V, K, dtype):
    test_logprob_and_gradients(N, V, K, dtype)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N", [1, 64, 65, 128])
def test_few_rows_keep_d_whole(N, dtype):
    h, w, t, g = inputs(N, 777, 96, dtype, seed=N)
    _, _, gh, gh_e, gw, gw_e = expect(h, w, t, g, dtype, parts=2)
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    a, b = torch.autograd.grad(sequence_log_probs_from_hidden(hd, wd, t.cuda()), [hd, wd], g.cuda())
    within(a.cpu(), gh, gh_e, "hidden's gradient")
    within(b.cpu(), gw, gw_e, "weight's gradient")


@pytest.mark.parametrize("N", [61, 100])
def test_few_rows_over_many_vocabulary_rows(N):
    """More of them per workgroup than it stages at once, a ragged end."""
    V, K = 30011, 4104
    h, w, t, g = (x.cuda() for x in inputs(N, V, K, BF, seed=N))
    lp, lp_e, gh, gh_e, gw, gw_e = expect(h, w, t, g, BF)
    h.requires_grad_(), w.requires_grad_()
    got = sequence_log_probs_from_hidden(h, w, t)
    within(got.detach(), lp, lp_e, "logprob")
    a, b = torch.autograd.grad(got, [h, w], g)
    within(a, gh, gh_e, "hidden's gradient")
    within(b, gw, gw_e, "weight's gradient")


def test_few_rows_beside_a_masked_vocabulary_row():
    """A vocabulary row of -inf logits takes no part, and the rows of the
    16-row blocks that are not there make no NaN of it."""
    for N in (5, 70):
        h, w, t, g = inputs(N, 40, 64, BF, seed=N)
        h = h.abs() + 0.5
        w[7], w[7, 3] = 0.0, float("-inf")
        t[t == 7] = 8
        keep = torch.arange(40) != 7
        small = torch.where(t > 7, t - 1, t)
        lp, lp_e, *_ = expect(h, w[keep], small, g, BF)
        hd, wd = h.cuda(), w.cuda().requires_grad_()
        got = sequence_log_probs_from_hidden(hd, wd, t.cuda())
        within(got.detach().cpu(), lp, lp_e, "logprob")
        (gw,) = torch.autograd.grad(got, [wd], g.cuda())
        assert bool((gw[7] == 0).all()) and bool(gw.isfinite().all())


@pytest.mark.parametrize("N", [3, 130])
def test_a_weight_past_32_bit_offsets(N):
    """Zero rows but a few: logits 0 there, so the sums are known."""
    V, K = (1 << 31) // 4096 + 777, 4096
    w = torch.zeros(V, K, dtype=BF, device="cuda")
    rows = torch.tensor([0, 1 << 19, V - 300, V - 1], device="cuda")
    g = torch.Generator().manual_seed(2)
    w[rows] = (torch.randn(4, K, generator=g) * 0.05).to(BF).cuda()
    h = torch.randn(N, K, generator=g).to(BF).cuda()
    t = rows[torch.arange(N, device="cuda") % 4]
    x = h.double() @ w[rows].double().T
    lse = torch.log(x.exp().sum(1) + (V - 4))
    grad = torch.linspace(0.5, 1.0, N, device="cuda")
    hd, wd = h.requires_grad_(), w.requires_grad_()
    lp = sequence_log_probs_from_hidden(hd, wd, t)
    want = x[torch.arange(N), torch.arange(N) % 4] - lse
    mag = (h.double().abs() @ w[rows].double().abs().T).amax(1)
    err = 2 * (K * W * mag + 4 * W * (1 + x.abs().amax(1))) + 64 * W + 2 * W * want.abs()
    within(lp.detach(), want.detach(), err.detach(), "logprob")
    gh, gw = torch.autograd.grad(lp, [hd, wd], grad)
    p = (x - lse[:, None]).exp().detach()
    d = -p * grad[:, None]
    d[torch.arange(N), torch.arange(N) % 4] += grad
    u = half_step(BF)
    d_err = u * d.abs() + (1 + u) * grad[:, None] * p * 2 * err.detach()[:, None] + 4 * W
    tiny = torch.finfo(BF).smallest_normal * torch.finfo(BF).eps / 2
    for got, a, e, b in ((gw[rows], d.T, d_err.T, h), (gh, d, d_err, w.detach()[rows])):
        b = b.detach().double()
        r = a @ b
        e = e @ b.abs() + (V + N) * W * ((a.abs() + e) @ b.abs())
        within(got, r, e + u * (r.abs() + e) + tiny, "gradient")
    # a zero row's gradient: -sum g_n h_n / exp(lse_n); D is off by u and by
    # twice the logprobs' error, the sum by N w, the result rounded once
    one = gw[V - 2].double()
    r = -(grad.double()[:, None] * h.detach().double() * (-lse.detach())[:, None].exp()).sum(0)
    mag = (grad.double()[:, None] * h.detach().double().abs() * (-lse.detach())[:, None].exp()).sum(0)
    rel = 2 * u + 2 * float(err.max()) + N * W
    within(one, r, rel * mag + tiny, "a zero row's gradient")


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_mean_loss_skips_ignored(dtype):
    B, S, V, K = 3, 90, 611, 96
    h, w, t, _ = inputs(B * S, V, K, dtype, seed=5)
    labels = t.view(B, S).clone()
    labels[:, 1:] = t.view(B, S)[:, :-1]
    labels[0, :40] = -100
    labels[2, 60:] = -100
    target = labels[:, 1:].reshape(-1)
    keep = target != -100
    rows = h.view(B, S, K)[:, :-1].reshape(-1, K)
    g = torch.where(keep, -1.0 / keep.sum(), 0.0)
    lp, lp_e, gh, gh_e, gw, gw_e = expect(rows, w, target.clamp(min=0), g, dtype)
    # ignored rows hold anything
    hd = h.view(B, S, K).clone()
    hd[:, :-1][~keep.view(B, S - 1)] = float("nan")
    hd = hd.cuda().requires_grad_()
    wd = w.cuda().requires_grad_()
    loss = sft_cross_entropy_loss_from_hidden(hd, wd, labels.cuda())
    want = -(lp[keep].sum() / keep.sum())
    assert abs(float(loss.detach()) - float(want)) <= float(lp_e[keep].mean()) + 2 * W * abs(float(want))
    a, b = torch.autograd.grad(loss, [hd, wd])
    assert bool((a[:, -1] == 0).all())
    a = a[:, :-1].reshape(-1, K)
    assert bool((a[~keep.cuda()] == 0).all())
    within(a.cpu()[keep], gh[keep], gh_e[keep], "hidden's gradient")
    within(b.cpu(), gw, gw_e, "weight's gradient")


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,S,drop", [(2, 41, 30), (1, 129, 5), (4, 2, 0), (3, 30, 86)])
def test_mean_loss_of_few_rows(B, S, drop, dtype):
    """`drop` of the B x (S - 1) positions ignored, at random."""
    V, K = 700, 72
    h, w, t, _ = inputs(B * (S - 1), V, K, dtype, seed=B + S)
    keep = torch.ones(B * (S - 1), dtype=torch.bool)
    keep[torch.randperm(B * (S - 1), generator=torch.Generator().manual_seed(1))[:drop]] = False
    labels = torch.zeros(B, S, dtype=torch.int64)
    labels[:, 1:] = torch.where(keep, t, -100).view(B, S - 1)
    g = torch.where(keep, -1.0 / keep.sum(), 0.0)
    lp, lp_e, gh, gh_e, gw, gw_e = expect(h, w, t, g, dtype, parts=2)
    hd = torch.full((B, S, K), float("nan"), dtype=dtype)
    hd[:, :-1] = torch.where(keep[:, None], h, torch.full_like(h, float("nan"))).view(B, S - 1, K)
    hd, wd = hd.cuda().requires_grad_(), w.cuda().requires_grad_()
    loss = sft_cross_entropy_loss_from_hidden(hd, wd, labels.cuda())
    want = -(lp[keep].sum() / keep.sum())
    assert abs(float(loss.detach()) - float(want)) <= float(lp_e[keep].mean()) + 2 * W * abs(float(want))
    a, b = torch.autograd.grad(loss, [hd, wd])
    assert bool((a[:, -1] == 0).all())
    a = a[:, :-1].reshape(-1, K).cpu()
    assert bool((a[~keep] == 0).all())
    # (the mean's gradient is divided and multiplied in fp32: 2 w more)
    more = 2 * W
    within(a[keep], gh[keep], (gh_e + more * gh.abs())[keep], "hidden's gradient")
    within(b.cpu(), gw, gw_e + more * gw.abs(), "weight's gradient")


def test_scaled_loss_gradient():
    """The loss's own gradient scales both gradients."""
    h, w, t, _ = inputs(50, 300, 64, BF, seed=9)
    hd, wd = h.cuda().view(1, 50, 64).requires_grad_(), w.cuda().requires_grad_()
    labels = t.cuda().view(1, 50)
    one = torch.autograd.grad(sft_cross_entropy_loss_from_hidden(hd, wd, labels), [hd, wd])
    four = torch.autograd.grad(sft_cross_entropy_loss_from_hidden(hd, wd, labels) * 4.0, [hd, wd])
    for a, b in zip(one, four):  # a power of two is exact everywhere
        assert torch.equal(a.float() * 4.0, b.float())


def test_no_row_left():
    h, w, t, _ = inputs(20, 100, 64, BF, seed=1)
    hd, wd = h.cuda().view(2, 10, 64).requires_grad_(), w.cuda().requires_grad_()
    labels = torch.full((2, 10), -100, device="cuda")
    loss = sft_cross_entropy_loss_from_hidden(hd, wd, labels)
    assert bool(loss.isnan())  # 0 / 0, as F.cross_entropy gives
    lp = sequence_log_probs_from_hidden(hd, wd, labels, ignore_index=-100)
    assert bool((lp == 0).all())
    for x in torch.autograd.grad(lp.sum(), [hd, wd]):
        assert bool((x == 0).all())
    for shape in ((0, 10), (2, 0)):
        e = torch.empty(*shape, 64, device="cuda", dtype=BF, requires_grad=True)
        lp = sequence_log_probs_from_hidden(e, wd, torch.empty(shape, dtype=torch.int64, device="cuda"))
        assert lp.shape == shape
        a, b = torch.autograd.grad(lp.sum(), [e, wd])
        assert a.shape == e.shape and bool((b == 0).all())


def test_single_position_has_no_target():
    h = torch.randn(4, 1, 64, device="cuda").to(BF).requires_grad_()
    w = torch.randn(50, 64, device="cuda").to(BF).requires_grad_()
    loss = sft_cross_entropy_loss_from_hidden(h, w, torch.zeros(4, 1, dtype=torch.int64, device="cuda"))
    assert bool(loss.isnan())
    a, b = torch.autograd.grad(loss, [h, w])
    assert bool((a == 0).all()) and bool((b == 0).all())


LAYOUTS = {
    "shifted": lambda h: torch.cat([h, h[:, :1]], 1)[:, :-1],
    "wide rows": lambda h: torch.cat([h, h], 2)[..., : h.shape[2]],
    "odd rows": lambda h: torch.nn.functional.pad(h, (0, 3))[..., : h.shape[2]],
    "columns apart": lambda h: h.transpose(1, 2).contiguous().transpose(1, 2),
    "batch inside": lambda h: h.transpose(0, 1).contiguous().transpose(0, 1),
    "one row for all": lambda h: h[:, :1].expand(h.shape),
}


@pytest.mark.parametrize("how", list(LAYOUTS))
def test_hidden_layouts(how):
    B, S, V, K = 2, 37, 400, 88
    h, w, t, g = inputs(B * S, V, K, BF, seed=11)
    base = LAYOUTS[how](h.view(B, S, K).cuda())
    hd, wd = base.detach().requires_grad_(), w.cuda().requires_grad_()
    if how != "columns apart":
        assert not hd.is_contiguous()
    plain = hd.detach().contiguous().requires_grad_()
    td = t.cuda().view(B, S)
    out = [sequence_log_probs_from_hidden(x, wd, td) for x in (hd, plain)]
    assert torch.equal(out[0], out[1])
    ga = torch.autograd.grad(out[0], [hd, wd], g.cuda().view(B, S))
    gb = torch.autograd.grad(out[1], [plain, wd], g.cuda().view(B, S))
    assert torch.equal(ga[0], gb[0]) and torch.equal(ga[1], gb[1])


@pytest.mark.parametrize("how", ["transposed", "wide rows", "unaligned", "odd rows"])
def test_weight_layouts(how):
    N, V, K = 70, 333, 64
    h, w, t, g = inputs(N, V, K, BF, seed=12)
    w = w.cuda()
    if how == "transposed":
        wd = w.t().contiguous().t()
    elif how == "wide rows":
        wd = torch.cat([w, w], 1)[:, :K]
    elif how == "unaligned":
        wd = torch.cat([w.new_zeros(1), w.reshape(-1)])[1:].view(V, K)
    else:
        wd = torch.nn.functional.pad(w, (0, 3))[:, :K]
    wd = wd.detach().requires_grad_()
    ws = w.clone().requires_grad_()
    hd, td = h.cuda().requires_grad_(), t.cuda()
    outs = []
    for x in (wd, ws):
        lp = sequence_log_probs_from_hidden(hd, x, td)
        outs.append((lp.detach(), *torch.autograd.grad(lp, [hd, x], g.cuda())))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_int32_and_strided_targets():
    B, S, V, K = 4, 21, 300, 64
    h, w, t, _ = inputs(B * S, V, K, HF, seed=13)
    hd, wd = h.cuda().view(B, S, K), w.cuda()
    want = sequence_log_probs_from_hidden(hd, wd, t.cuda().view(B, S))
    for ids in (t.int().cuda().view(B, S), t.cuda().view(B, S).t().contiguous().t(),
                torch.stack([t, t], 1).cuda()[:, 0].view(B, S)):
        assert torch.equal(sequence_log_probs_from_hidden(hd, wd, ids), want)


def test_rows_do_not_depend_on_ignored_ones():
    """Leaving rows out changes nothing for those that stay: their logprobs
    and hidden gradients keep their bits at any place in the list."""
    N, V, K = 300, 900, 64
    h, w, t, g = inputs(N, V, K, BF, seed=14)
    g = g.abs() + 0.1
    hd, wd, td = h.cuda().requires_grad_(), w.cuda(), t.cuda()
    full = sequence_log_probs_from_hidden(hd, wd, td)
    (gf,) = torch.autograd.grad(full, [hd], g.cuda())
    drop = torch.arange(N, device="cuda") % 3 == 0
    part = sequence_log_probs_from_hidden(hd, wd, torch.where(drop, -7, td), ignore_index=-7)
    (gp,) = torch.autograd.grad(part, [hd], g.cuda())
    assert torch.equal(part[~drop], full[~drop].detach()) and bool((part[drop] == 0).all())
    assert torch.equal(gp[~drop], gf[~drop]) and bool((gp[drop] == 0).all())


def test_only_what_is_asked_for():
    h, w, t, g = inputs(90, 500, 64, BF, seed=15)
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    lp = sequence_log_probs_from_hidden(hd, wd, t.cuda())
    both = torch.autograd.grad(lp, [hd, wd], g.cuda())
    lp = sequence_log_probs_from_hidden(hd, wd.detach(), t.cuda())
    assert torch.equal(torch.autograd.grad(lp, [hd], g.cuda())[0], both[0])
    lp = sequence_log_probs_from_hidden(hd.detach(), wd, t.cuda())
    assert torch.equal(torch.autograd.grad(lp, [wd], g.cuda())[0], both[1])


def test_fp16_small_gradients_keep_their_bits():
    """g of 1e-7 would leave fp16's numbers without the power of two in D."""
    N, V, K = 40, 3000, 64
    h, w, t, g = inputs(N, V, K, HF, seed=16)
    g = g * 1e-7
    hd, wd, td = h.cuda()[None], w.cuda(), t.cuda()[None]
    lse = ops.linear_logprob(hd, wd, td).lse
    # with an exponent at which the fp16 results have their bits, and at 1e-7
    # where they lie on fp16's smallest steps
    for k in (2.0 ** 20, 1.0):
        a, b = ops.linear_logprob_backward(hd, wd, td, lse, g.cuda()[None] * k)
        _, _, gh, gh_e, gw, gw_e = expect(h, w, t, g * k, HF)
        within(a[0].cpu(), gh, gh_e, "hidden's gradient")
        within(b.cpu(), gw, gw_e, "weight's gradient")


def test_large_and_infinite_logits():
    K = 64
    h = torch.zeros(4, K, dtype=BF)
    w = torch.zeros(300, K, dtype=BF)
    w[7, 0], w[8, 0] = 1.0, -1.0
    h[0, 0], h[1, 0] = 30000.0, -30000.0
    h[2, 0] = float("inf")
    h[3, 0] = float("nan")
    t = torch.tensor([7, 7, 0, 0])
    lp = sequence_log_probs_from_hidden(h.cuda(), w.cuda(), t.cuda()).cpu()
    # (bf16 has steps of 128 there: 30000 is 234 * 128 = 29952)
    assert float(lp[0]) == 0.0 and float(lp[1]) == -2 * 29952.0
    assert bool(lp[2].isnan()) and bool(lp[3].isnan())


def test_pieces_of_the_vocabulary():
    """More than one piece (a piece's gradient takes at most 1 GiB)."""
    N, V, K = 4200, 140001, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn(V, K, generator=gen, device="cuda") * 2 / K ** 0.5).to(BF)
    t = torch.randint(0, V, (N,), generator=gen, device="cuda")
    h = (torch.randn(N, K, generator=gen, device="cuda") + w[t].float()).to(BF)
    g = torch.randn(N, generator=gen, device="cuda")
    assert 2 * N * V > 1 << 30
    lp, lp_e, gh, gh_e, gw, gw_e = expect(h, w, t, g, BF)
    hd, wd = h.requires_grad_(), w.requires_grad_()
    got = sequence_log_probs_from_hidden(hd, wd, t)
    a, b = torch.autograd.grad(got, [hd, wd], g)
    within(got.detach(), lp, lp_e, "logprob")
    within(a, gh, gh_e, "hidden's gradient")
    within(b, gw, gw_e, "weight's gradient")
    again = torch.autograd.grad(sequence_log_probs_from_hidden(hd, wd, t), [hd, wd], g)
    assert torch.equal(a, again[0]) and torch.equal(b, again[1])


def test_memory_is_bounded_by_a_piece():
    N, V, K = 8192, 151936, 64
    h = torch.randn(N, K, device="cuda").to(BF).requires_grad_()
    w = torch.randn(V, K, device="cuda").to(BF).requires_grad_()
    t = torch.randint(0, V, (N,), device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    lp = sequence_log_probs_from_hidden(h, w, t)
    assert torch.cuda.memory_allocated() - before < 1 << 20  # kept for the backward
    lp.sum().backward()
    # the logits in 16 bits alone would take 2.5 GB
    assert torch.cuda.max_memory_allocated() - before < 1200 << 20


def test_other_stream():
    h, w, t, g = inputs(128, 700, 64, BF, seed=17)
    hd, wd, td, gd = h.cuda().requires_grad_(), w.cuda().requires_grad_(), t.cuda(), g.cuda()
    want = torch.autograd.grad(sequence_log_probs_from_hidden(hd, wd, td), [hd, wd], gd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = torch.autograd.grad(sequence_log_probs_from_hidden(hd, wd, td), [hd, wd], gd)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_and_replayed():
    """Forward and backward in one graph, replayed on new values with eager
    work between: each replay gives the eager bits."""
    N, V, K = 100, 520, 64
    gen = torch.Generator().manual_seed(18)
    h = torch.zeros(1, N, K, dtype=BF, device="cuda")
    w = torch.zeros(V, K, dtype=BF, device="cuda")
    t = torch.zeros(1, N, dtype=torch.int64, device="cuda")
    g = torch.zeros(1, N, device="cuda")

    def fill(k):
        a, b, c, d = inputs(N, V, K, BF, seed=100 + k)
        c[torch.rand(N, generator=gen) < 0.3] = -100
        h.copy_(a[None]), w.copy_(b), t.copy_(c[None]), g.copy_(d[None])

    def step():
        out = ops.linear_logprob(h, w, t, ignore_index=-100, mean=True)
        return (out.logprob, out.mean_loss, out.count,
                *ops.linear_logprob_backward(h, w, t, out.lse, g, ignore_index=-100))

    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        fill(k)
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
    # a bad target: nothing waits for it in a replay, its logprob is NaN
    t[0, 3] = V
    graph.replay()
    torch.cuda.synchronize()
    assert bool(held[0][0, 3].isnan()) and bool(held[1].isnan())


def test_labels_may_change_before_the_backward():
    h, w, t, _ = inputs(40, 300, 64, BF, seed=19)
    hd, wd = h.cuda().view(1, 40, 64).requires_grad_(), w.cuda().requires_grad_()
    labels = t.cuda().view(1, 40)
    want = torch.autograd.grad(sft_cross_entropy_loss_from_hidden(hd, wd, labels), [hd, wd])
    buf = labels.clone()
    loss = sft_cross_entropy_loss_from_hidden(hd, wd, buf)
    buf.zero_()
    got = torch.autograd.grad(loss, [hd, wd])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("bad", [-1, 300, 2 ** 31, -2 ** 40])
def test_bad_target_raises(bad):
    h, w, t, _ = inputs(30, 300, 64, BF, seed=20)
    t[17] = bad
    with pytest.raises(RuntimeError, match="outside"):
        sequence_log_probs_from_hidden(h.cuda(), w.cuda(), t.cuda())
    with pytest.raises(RuntimeError, match="outside"):
        sft_cross_entropy_loss_from_hidden(h.cuda()[None], w.cuda(), t.cuda()[None])
    # ignored, it is not bad
    assert float(sequence_log_probs_from_hidden(h.cuda(), w.cuda(), t.cuda(), ignore_index=bad)[17]) == 0.0
