"""The operators of a training step around the vocabulary matrix, as measurable cases.

A step with hidden states at both ends looks tokens up in the embedding, runs
the model, turns the last hidden states into token losses or logprobs through
the lm_head, and clips the gradients before the optimizer.  The operators are
the parts of it whose size is the vocabulary's or the model's:

- ``logprobs`` / ``sft``: token logprobs or the mean cross entropy from hidden
  states and the lm_head weight, in pieces of the vocabulary, without keeping
  the logits, with the gradients of both
  (``sequence_log_probs_from_hidden``, ``sft_cross_entropy_loss_from_hidden``).
- ``embed``: the embedding lookup with its scale, and the gradient of the
  table by sorted tokens (``token_embedding``).
- ``clip``: the global norm of the gradients of many tensors, and their
  clipping (``clip_grad_norm_``).

``own`` picks the framework's calls; without it ``run`` computes the same by
elementary operations.  A case is a dict of plain values.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100


def listed():
    return [
        # a step on the policy's own rollouts at the largest size the hidden
        # path is benchmarked on: per-token logprobs, and their gradient from
        # the loss's gradient per token (zero behind each sequence's end)
        dict(name="policy_long", kind="logprobs", grad=True, batch=4, seq=2048, width=4096,
             vocab=248320, dtype="bf16"),
        # a supervised step: mean loss over the completions, prompts ignored
        dict(name="sft_step", kind="sft", grad=True, batch=8, seq=512, width=4096, vocab=151936,
             dtype="bf16"),
        # a small fp16 policy step, odd vocabulary and odd number of tokens
        dict(name="policy_ragged", kind="logprobs", grad=True, batch=3, seq=333, width=2816,
             vocab=50257, dtype="fp16"),
        # one short completion with its gradient
        dict(name="policy_short", kind="logprobs", grad=True, batch=1, seq=61, width=4096,
             vocab=151936, dtype="bf16"),
        # scoring without a gradient, as old logprobs are computed
        dict(name="score_fp16", kind="logprobs", grad=False, batch=2, seq=1024, width=4096,
             vocab=151936, dtype="fp16"),
        # the embedding of one decode step of a group of 64: latency
        dict(name="embed_decode", kind="embed", grad=False, batch=64, seq=1, width=4096,
             vocab=151936, dtype="bf16", scale=1.0, pad=-1),
        # the embedding of a training batch with right padding and its
        # table's gradient
        dict(name="embed_train", kind="embed", grad=True, batch=8, seq=1024, width=4096,
             vocab=151936, dtype="bf16", scale=64.0, pad=0),
        # the same in fp32, with an odd width, an odd vocabulary
        dict(name="embed_ragged", kind="embed", grad=True, batch=3, seq=333, width=1027,
             vocab=50257, dtype="fp32", scale=1.0, pad=-1),
        # the gradients of low-rank adapters: 504 small fp32 tensors, the
        # views of one bucket
        dict(name="clip_adapters", kind="clip", tensors="adapters", layers=36, width=4096,
             rank=16, vocab=0, dtype="fp32", max_norm=1.0, norm="2"),
        # the bf16 gradients of a whole model with its vocabulary matrix
        dict(name="clip_model", kind="clip", tensors="layers", layers=8, width=4096, rank=0,
             vocab=151936, dtype="bf16", max_norm=1.0, norm="2"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _vocab(rng):
    v = _log_int(rng, 32000, 248320)
    # most lm_heads are padded to a multiple of 64; some vocabularies are odd
    return v if rng.random() < 0.3 else min(248320, (v + 63) // 64 * 64)


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "sft", "embed", "embed", "clip"])
    if kind in ("logprobs", "sft"):
        b = rng.choice([1, 2, 3, 4])
        # widths of models, now and then one that is no multiple of 128
        width = 128 * rng.randint(4, 32) if rng.random() < 0.8 else 8 * rng.randint(64, 511)
        return dict(kind=kind, grad=kind == "sft" or rng.random() < 0.7, batch=b,
                    seq=max(2, _log_int(rng, 8, 8192) // b), width=width, vocab=_vocab(rng),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "embed":
        grad = rng.random() < 0.7
        n = _log_int(rng, 1, 32768)
        b = max(1, min(n, rng.choice([1, 2, 3, 8])))
        width = 128 * rng.randint(4, 32) if rng.random() < 0.8 else rng.randint(500, 4096)
        return dict(kind=kind, grad=grad, batch=b, seq=max(1, n // b), width=width,
                    vocab=_vocab(rng), dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"]),
                    scale=rng.choice([1.0, 1.0, math.sqrt(width)]), pad=rng.choice([-1, 0]))
    adapters = rng.random() < 0.5
    return dict(kind=kind, tensors="adapters" if adapters else "layers",
                layers=rng.randint(2, 36) if adapters else rng.randint(1, 6),
                width=64 * rng.randint(8, 64), rank=rng.choice([8, 16, 32]) if adapters else 0,
                vocab=0 if adapters else _vocab(rng),
                dtype=rng.choice(["fp32", "bf16", "fp32", "fp16"]),
                max_norm=rng.choice([0.5, 1.0, 1.0, 1e4]), norm=rng.choice(["2", "2", "2", "inf"]))


# ------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _weight(V, H, dtype, g, spread):
    """A [V, H] table of normal rows whose norm is about ``spread``."""
    w = torch.empty((V, H), dtype=dtype, device="cuda")
    for s in range(0, V, 32768):
        w[s : s + 32768] = torch.randn((min(32768, V - s), H), generator=g, device="cuda").mul_(
            spread / math.sqrt(H))
    return w


def _shapes(case):
    """The shapes of the tensors whose gradients are clipped."""
    d, r = case["width"], case["rank"]
    ffn = 11 * d // 4
    linears = [(d, d), (d // 4, d), (d // 4, d), (d, d), (ffn, d), (ffn, d), (d, ffn)]
    out = []
    for _ in range(case["layers"]):
        for o, i in linears:
            out += [(r, i), (o, r)] if case["tensors"] == "adapters" else [(o, i)]
        if case["tensors"] == "layers":
            out += [(d,), (d,)]
    if case["vocab"]:
        out += [(case["vocab"], d), (d,)]
    return out


def _likely_ids(n, V, g):
    """Ids whose frequency falls with their number, as a vocabulary's does:
    id 0 takes a few percent of the tokens, most ids none."""
    u = torch.rand((n,), generator=g, device="cuda", dtype=torch.float64)
    return (u.mul_(math.log(V + 1.0)).exp_() - 1.0).to(torch.int64).clamp_(0, V - 1)


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "clip":
        dt = DTYPES[case["dtype"]]
        shapes = _shapes(case)
        total = sum(math.prod(s) for s in shapes)
        fresh = torch.empty((total,), dtype=dt, device="cuda")
        # gradients of differing sizes: a factor of up to 30 between tensors
        scale = (torch.rand((len(shapes),), generator=g, device="cuda") * 3.4).exp_()
        scale = scale.mul_(2e-3 if case["tensors"] == "adapters" else 1e-4).tolist()
        grads = torch.empty_like(fresh)
        data = torch.zeros_like(fresh)
        params, at = [], 0
        for s, k in zip(shapes, scale):
            n = math.prod(s)
            for a in range(at, at + n, 1 << 27):
                m = min(1 << 27, at + n - a)
                fresh[a : a + m] = torch.randn((m,), generator=g, device="cuda").mul_(k)
            p = torch.nn.Parameter(data[at : at + n].view(s))
            p.grad = grads[at : at + n].view(s)
            params.append(p)
            at += n
        return dict(case=case, fresh=fresh, grads=grads, params=params)
    B, S, V, H = case["batch"], case["seq"], case["vocab"], case["width"]
    n, dt = B * S, DTYPES[case["dtype"]]
    if kind == "embed":
        ids = _likely_ids(n, V, g).view(B, S)
        if case["pad"] >= 0 and S > 1:
            ends = torch.randint(max(1, S // 2), S + 1, (B, 1), generator=g, device="cuda")
            ids[torch.arange(S, device="cuda").unsqueeze(0) >= ends] = case["pad"]
        st = dict(case=case, ids=ids, weight=_weight(V, H, dt, g, 1.0))
        if case["grad"]:
            st["weight"].requires_grad_(True)
            st["g"] = torch.randn((B, S, H), generator=g, device="cuda").mul_(1e-3).to(dt)
        return st
    # normalised hidden states and a weight whose logits spread by about 2; a
    # token's hidden state leans to its own target's weight row
    hid = torch.randn((n, H), generator=g, device="cuda")
    w = _weight(V, H, dt, g, 2.0)
    t = torch.randint(0, V, (n,), generator=g, device="cuda")
    lean = torch.rand((n, 1), generator=g, device="cuda") * 3.0
    hid = (hid + w[t].float() * lean).to(dt).view(B, S, H)
    ids = t.view(B, S)
    st = dict(case=case, hidden=hid, weight=w, ids=ids)
    if kind == "sft":
        # labels[:, 1:] are the targets of the positions before them
        labels = torch.full_like(ids, IGNORE)
        labels[:, 1:] = ids[:, :-1]
        prompt = torch.randint(1, max(2, S // 2), (B, 1), generator=g, device="cuda")
        labels[torch.arange(S, device="cuda").unsqueeze(0) < prompt] = IGNORE
        st["labels"] = labels
    elif case["grad"]:
        # the loss's gradient per token: an advantage per sequence, a ratio
        # near 1, zero behind the sequence's end
        adv = torch.randn((B, 1), generator=g, device="cuda")
        ratio = 1.0 + 0.1 * torch.randn((B, S), generator=g, device="cuda")
        ends = torch.randint(max(1, S // 2), S + 1, (B, 1), generator=g, device="cuda")
        live = torch.arange(S, device="cuda").unsqueeze(0) < ends
        st["g"] = torch.where(live, -adv * ratio / (ends * B), 0.0)
    if case["grad"]:
        hid.requires_grad_(True)
        w.requires_grad_(True)
    return st


# --------------------------------------------------------------------- runs

def _own(state):
    c = state["case"]
    if c["kind"] == "clip":
        from graspo_amd.grad_clip import clip_grad_norm_

        state["grads"].copy_(state["fresh"])  # a backward's new gradients
        norm = clip_grad_norm_(state["params"], c["max_norm"], norm_type=float(c["norm"]))
        return norm, state["grads"]
    if c["kind"] == "embed":
        from graspo_amd.embedding import token_embedding

        # a decode loop's ids come from the sampler: it does not wait for a
        # look at them
        out = token_embedding(state["ids"], state["weight"], scale=c["scale"],
                              padding_idx=c["pad"] if c["pad"] >= 0 else None,
                              check_status=c["grad"])
        if not c["grad"]:
            return out
        return out.detach(), *torch.autograd.grad(out, [state["weight"]], state["g"])
    h, w = state["hidden"], state["weight"]
    if c["kind"] == "sft":
        from graspo_amd.sft_loss import sft_cross_entropy_loss_from_hidden

        loss = sft_cross_entropy_loss_from_hidden(h, w, state["labels"], ignore_index=IGNORE)
        return loss.detach(), *torch.autograd.grad(loss, [h, w])
    from graspo_amd.graspo_loss import sequence_log_probs_from_hidden

    lp = sequence_log_probs_from_hidden(h, w, state["ids"])
    if not c["grad"]:
        return lp
    return lp.detach(), *torch.autograd.grad(lp, [h, w], state["g"])


def _plain_logprobs(h, w, t, g, want_grad):
    """(log_softmax(h w^T)[t], gradients of both) of rows h [N, H] in 32 bits;
    ``g``: what each row's logprob is weighted with, or a function of them."""
    x = h @ w.t()
    top = x.amax(1, keepdim=True)
    e = (x - top).exp_()
    s = e.sum(1, keepdim=True)
    lp = x.gather(1, t.unsqueeze(1)) - top - s.log()
    del x
    if not want_grad:
        return lp.squeeze(1), None, None
    g = g.unsqueeze(1)
    d = e.mul_(-g / s)
    d.scatter_add_(1, t.unsqueeze(1), g)
    return lp.squeeze(1), d @ w, d.t() @ h


@torch.no_grad()
def _plain(state):
    c = state["case"]
    if c["kind"] == "clip":
        grads = state["grads"]
        grads.copy_(state["fresh"])
        x = grads.float()
        if c["norm"] == "inf":
            norm = x.abs().amax()
        else:
            norm = x.to(torch.float64).square_().sum().sqrt().float()
        coef = (c["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        grads.copy_(x.mul_(coef))
        return norm, grads
    if c["kind"] == "embed":
        w, ids = state["weight"], state["ids"]
        out = (w[ids].float() * c["scale"]).to(w.dtype)
        if not c["grad"]:
            return out
        rows = state["g"].float() * c["scale"]
        if c["pad"] >= 0:
            rows = rows * (ids != c["pad"]).unsqueeze(-1)
        acc = torch.zeros(w.shape, dtype=torch.float32, device="cuda")
        acc.index_add_(0, ids.reshape(-1), rows.reshape(-1, w.shape[1]))
        return out, acc.to(w.dtype)
    h, w = state["hidden"], state["weight"]
    B, S, H = h.shape
    if c["kind"] == "sft":
        t = torch.full_like(state["labels"], IGNORE)
        t[:, :-1] = state["labels"][:, 1:]
        live = t != IGNORE
        g = live.float() / -live.sum()
        lp, gh, gw = _plain_logprobs(h.reshape(-1, H).float(), w.float(),
                                     t.clamp(min=0).reshape(-1), g.reshape(-1), True)
        first = (lp * g.reshape(-1)).sum()
    else:
        g = state["g"].reshape(-1) if c["grad"] else None
        lp, gh, gw = _plain_logprobs(h.reshape(-1, H).float(), w.float(),
                                     state["ids"].reshape(-1), g, c["grad"])
        first = lp.view(B, S)
        if not c["grad"]:
            return first
    return first, gh.view(B, S, H).to(h.dtype), gw.to(w.dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------ what it needs

def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": 2 * n * size, "flops": 3 * n}
    n, V, H = case["batch"] * case["seq"], case["vocab"], case["width"]
    if kind == "embed":
        rows = min(n, V)
        b = 8 * n + (rows + n) * H * size
        if case["grad"]:
            b += n * H * size + V * H * size
        return {"bytes": b, "flops": (2 if case["grad"] else 1) * n * H}
    b = (n * H + V * H) * size + n * 12
    f = 2 * n * H * V
    # with gradients: both operands' gradients written, two more products
    return {"bytes": 2 * b, "flops": 3 * f} if case["grad"] else {"bytes": b, "flops": f}


# ------------------------------------------------------------- in 64 bits

@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    if kind == "clip":
        parts = [p.grad for p in st["params"]]
        at, powers = 0, []
        for q in parts:
            x = st["fresh"][at : at + q.numel()].to(f64)
            powers.append(x.abs().max() if case["norm"] == "inf" else torch.dot(x, x))
            at += q.numel()
        powers = torch.stack(powers)
        norm = powers.max() if case["norm"] == "inf" else powers.sum().sqrt()
        factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        return norm, st["fresh"].to(f64).mul_(factor)
    if kind == "embed":
        w, ids = st["weight"].detach(), st["ids"]
        out = torch.nn.functional.embedding(ids, w.to(f64)) * case["scale"]
        if not case["grad"]:
            return out
        flat, order = torch.sort(ids.reshape(-1), stable=True)
        rows = st["g"].reshape(-1, w.shape[1])[order].to(f64)
        grad = torch.zeros(w.shape, dtype=f64, device="cuda")
        uniq, counts = torch.unique_consecutive(flat, return_counts=True)
        ends = counts.cumsum(0)
        for part in range(0, w.shape[1], 1024):
            run_sum = rows[:, part : part + 1024].cumsum(0)
            upto = run_sum[ends - 1]
            upto[1:] -= run_sum[ends[:-1] - 1]
            grad[uniq, part : part + 1024] = upto * case["scale"]
        if case["pad"] >= 0:
            grad[case["pad"]] = 0.0
        return out, grad
    h, w = st["hidden"].detach(), st["weight"].detach().to(f64)
    B, S, H = h.shape
    rows = h.reshape(-1, H)
    if kind == "sft":
        t = torch.nn.functional.pad(st["labels"][:, 1:], (0, 1), value=IGNORE).reshape(-1)
        keep = (t != IGNORE).to(f64)
        weight_of = keep / keep.sum()
    else:
        t = st["ids"].reshape(-1)
        weight_of = -st["g"].reshape(-1).to(f64) if case["grad"] else None
    lps = []
    gh = torch.empty((rows.shape[0], H), dtype=f64, device="cuda")
    gw = torch.zeros(w.shape, dtype=f64, device="cuda") if case["grad"] else None
    for a in range(0, rows.shape[0], 1024):
        hb, tb = rows[a : a + 1024].to(f64), t[a : a + 1024].clamp(min=0)
        logits = torch.matmul(hb, w.t())
        logits -= torch.logsumexp(logits, dim=1, keepdim=True)
        at = torch.arange(tb.numel(), device="cuda")
        lps.append(logits[at, tb])
        if case["grad"]:
            prob = logits.exp_()
            prob[at, tb] -= 1.0
            prob *= weight_of[a : a + 1024, None]
            gh[a : a + 1024] = torch.matmul(prob, w)
            gw += torch.matmul(prob.t(), hb)
    lp = torch.cat(lps)
    if kind == "sft":
        return -(lp * weight_of).sum(), gh.view(B, S, H), gw
    if not case["grad"]:
        return lp.view(B, S)
    return lp.view(B, S), gh.view(B, S, H), gw
