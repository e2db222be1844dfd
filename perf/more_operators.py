"""The operators of a rollout of many requests, as measurable cases.

A batch of requests, each with its own low-rank adapter, is searched with
beams: every projection adds the requests' adapters, the logits of all beams
go through one selection, and the models' states follow the beams.  The same
adapters are what a training step learns.

- ``beam``: one step of a beam search over ``[groups * beams, vocab]`` logits:
  the best candidates over beams and vocabulary, the finished ones into each
  group's pool, the others into the beams' slots (``beam_step``).
- ``reorder`` / ``expand``: the states of all layers moved to the beams that
  go on, in place, or a prompt's states given to each of its beams
  (``reorder_states_``, ``expand_states``).
- ``lora``: low-rank adapters beside a shared projection, a request's own or
  none, with the gradients (``lora_add``).

``own`` picks the framework's calls; without it ``run`` computes the same by
elementary operations.  A case is a dict of plain values.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
          "uint8": torch.uint8}
PAD = 0


def listed():
    return [
        # one request with 4 beams, a step in the middle: latency
        dict(name="beam_one", kind="beam", groups=1, beams=4, vocab=151936, dtype="bf16",
             masked=False, first=False, step=17, penalty=1.0, early=False),
        # the largest batch of rows that the sampler is benchmarked on
        dict(name="beam_full", kind="beam", groups=32, beams=8, vocab=248320, dtype="bf16",
             masked=False, first=False, step=200, penalty=1.0, early=False),
        # a structured answer: a quarter of an odd vocabulary allowed, fp32 logits
        dict(name="beam_masked", kind="beam", groups=5, beams=3, vocab=50257, dtype="fp32",
             masked=True, first=False, step=33, penalty=0.6, early=True),
        # the first step behind the prompts: one live beam in each group
        dict(name="beam_first", kind="beam", groups=8, beams=5, vocab=151936, dtype="fp16",
             masked=False, first=True, step=0, penalty=1.0, early=False),
        # one request's cache of a short prompt, 28 layers: latency
        dict(name="reorder_short", kind="reorder", groups=1, beams=4, dead=2, layers=28, heads=8,
             dim=128, length=61, room=128, dtype="bf16"),
        # long prompts of a batch: 3 of 8 beams replaced
        dict(name="reorder_long", kind="reorder", groups=4, beams=8, dead=3, layers=8, heads=8,
             dim=128, length=4001, room=4096, dtype="bf16"),
        # behind a prefill: each prompt's cache for each of its beams
        dict(name="expand", kind="expand", groups=8, beams=4, dead=0, layers=12, heads=4, dim=128,
             length=999, room=999, dtype="bf16"),
        # one request's token through one projection: latency
        dict(name="lora_token", kind="lora", grad=False, batch=1, seq=1, width=4096, out=4096,
             rank=16, adapters=1, none=0, dtype="bf16"),
        # a decode step of 64 requests with 8 adapters, some with none
        dict(name="lora_decode", kind="lora", grad=False, batch=64, seq=1, width=4096, out=11264,
             rank=16, adapters=8, none=7, dtype="bf16"),
        # a training step of one adapter with its gradients
        dict(name="lora_train", kind="lora", grad=True, batch=8, seq=1024, width=4096, out=4096,
             rank=16, adapters=1, none=0, dtype="bf16"),
        # several adapters trained at once, ragged sizes
        dict(name="lora_ragged", kind="lora", grad=True, batch=6, seq=333, width=2816, out=1027,
             rank=8, adapters=5, none=1, dtype="fp16"),
        # the same in fp32 with a larger rank
        dict(name="lora_fp32", kind="lora", grad=True, batch=4, seq=500, width=2048, out=5632,
             rank=64, adapters=2, none=0, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["beam", "beam", "reorder", "expand", "lora", "lora", "lora"])
    if kind == "beam":
        beams = rng.choice([2, 3, 4, 5, 8, 16])
        vocab = _log_int(rng, 32000, 248320)
        # most vocabularies of logits are padded to a multiple of 64
        vocab = vocab if rng.random() < 0.3 else min(248320, (vocab + 63) // 64 * 64)
        first = rng.random() < 0.15
        return dict(kind=kind, groups=_log_int(rng, 1, 256 // beams), beams=beams, vocab=vocab,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    masked=rng.random() < 0.3, first=first,
                    step=0 if first else _log_int(rng, 1, 2000),
                    penalty=rng.choice([1.0, 1.0, 0.0, 0.6, 1.3]), early=rng.random() < 0.3)
    if kind in ("reorder", "expand"):
        beams = rng.choice([2, 3, 4, 5, 8, 16])
        groups = rng.randint(1, max(1, 32 // beams))
        layers, heads = rng.randint(1, 16), rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 128, 128, 256])
        # at most 4.2 GB in all
        most = int(4.2e9 / (2 * layers * heads * dim * 4 * groups * beams))
        length = _log_int(rng, 1, min(8192, most))
        room = min(most, (length + 127) // 128 * 128) if rng.random() < 0.6 else length
        return dict(kind=kind, groups=groups, beams=beams,
                    dead=rng.randint(0 if beams == 2 else 1, beams - 1) if kind == "reorder" else 0,
                    layers=layers, heads=heads, dim=dim, length=length, room=max(length, room),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32", "uint8"]))
    grad = rng.random() < 0.5
    rows = _log_int(rng, 1, 8192)
    # rows of whole sequences, or one token of each request
    batch = rng.choice([1, 2, 3, 8]) if rows >= 8 and (grad or rng.random() < 0.5) else \
        min(rows, 256)
    adapters = rng.choice([1, 1, 2, 3, 5, 8, 16])
    size = lambda: 128 * rng.randint(4, 32) if rng.random() < 0.8 else rng.randint(500, 4096)  # noqa: E731
    return dict(kind=kind, grad=grad, batch=batch, seq=max(1, rows // batch), width=size(),
                out=size(), rank=rng.choice([4, 8, 8, 16, 16, 32, 64]), adapters=adapters,
                none=rng.choice([0, 0, batch // 4]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


# ------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(shape, g):
    return torch.rand(shape, generator=g, device="cuda")


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _prepare_beam(case, g):
    G, K, V, dt = case["groups"], case["beams"], case["vocab"], DTYPES[case["dtype"]]
    logits = torch.empty((G * K, V), dtype=dt, device="cuda")
    for r in range(0, G * K, 32):
        logits[r : r + 32] = _randn((min(32, G * K - r), V), g).mul_(2.5)
    # a few likely tokens in each row, as a model's logits have
    likely = torch.randint(1, V, (G * K, 6), generator=g, device="cuda")
    logits.scatter_add_(1, likely, (6.0 + 6.0 * _rand((G * K, 6), g)).to(dt))
    eos = V - 3
    ends = _rand((G * K,), g) < 0.15
    logits[:, eos] = torch.where(ends, (14.0 + _rand((G * K,), g)).to(dt), logits[:, eos])
    inf = float("inf")
    if case["first"]:
        scores = torch.full((G, K), -inf, device="cuda")
        scores[:, 0] = 0.0
    else:
        scores = -(0.2 + _rand((G, K), g)) * math.sqrt(case["step"] + 1.0) - 2.0 * _rand((G, 1), g)
    t = case["step"]
    # finished hypotheses of earlier steps, best first, and groups that are done
    filled = torch.randint(0, (K + 1) if t else 1, (G, 1), generator=g, device="cuda")
    has = torch.arange(K, device="cuda").unsqueeze(0) < filled
    pool = (-(0.3 + _rand((G, K), g))).sort(dim=1, descending=True).values
    steps = torch.randint(0, max(t, 1), (G, K), generator=g, device="cuda", dtype=torch.int32)
    rows = torch.randint(0, K, (G, K), generator=g, device="cuda", dtype=torch.int32)
    rows += K * torch.arange(G, device="cuda", dtype=torch.int32).unsqueeze(1)
    done = (_rand((G,), g) < 0.1) & (torch.arange(G, device="cuda") > 0) & (t > 0)
    st = dict(case=case, logits=logits, scores=scores, eos=eos,
              pool_scores=torch.where(has, pool, -inf), pool_rows=torch.where(has, rows, -1),
              pool_steps=torch.where(has, steps, -1), done=done, mask=None)
    if case["masked"]:
        words = (V + 31) // 32
        bits = [torch.randint(-2**31, 2**31, (G * K, words), generator=g, device="cuda",
                              dtype=torch.int32) for _ in range(2)]
        st["mask"] = bits[0] & bits[1]
    return st


def _parents(G, K, dead, seed):
    """Rows that take over others: `dead` slots of each group continue one of
    the others, which keep their slots."""
    rng = random.Random(seed)
    out = []
    for b in range(G):
        gone = set(rng.sample(range(K), dead))
        kept = [k for k in range(K) if k not in gone]
        out += [b * K + (rng.choice(kept) if k in gone else k) for k in range(K)]
    return out


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "beam":
        return _prepare_beam(case, g)
    if kind in ("reorder", "expand"):
        G, K = case["groups"], case["beams"]
        R = G * K if kind == "reorder" else G
        shape = (2 * case["layers"], R, case["heads"], case["room"], case["dim"])
        cache = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda")
        for i in range(shape[0]):
            cache[i] = torch.randint(0, 256, shape[1:], generator=g, device="cuda",
                                     dtype=torch.uint8) if case["dtype"] == "uint8" else \
                _randn(shape[1:], g)
        live = cache[:, :, :, : case["length"]]
        st = dict(case=case, cache=cache, states=list(live.unbind(0)), live=live)
        if kind == "reorder":
            st["parents"] = torch.tensor(_parents(G, K, case["dead"], seed), dtype=torch.int32,
                                         device="cuda")
        return st
    B, S, K, N = case["batch"], case["seq"], case["width"], case["out"]
    E, r, dt = case["adapters"], case["rank"], DTYPES[case["dtype"]]
    # what the shared projection gave, and the inputs that it had
    st = dict(case=case, base=_randn((B, S, N), g).to(dt), x=_randn((B, S, K), g).to(dt),
              a=_randn((E, r, K), g).mul_(1.0 / math.sqrt(K)).to(dt),
              b=_randn((E, N, r), g).mul_(0.1).to(dt),
              scaling=0.5 + 1.5 * _rand((E,), g))
    ids = torch.randint(0, E, (B,), generator=g, device="cuda", dtype=torch.int32)
    ids[torch.randperm(B, generator=g, device="cuda")[: min(case["none"], B - 1)]] = -1
    st["ids"] = ids
    if case["grad"]:
        st["g"] = _randn((B, S, N), g).mul_(1e-3).to(dt)
        for k in ("x", "a", "b"):
            st[k].requires_grad_(True)
    return st


# --------------------------------------------------------------------- runs

def _own(state):
    c = state["case"]
    if c["kind"] == "beam":
        from graspo_amd.beam_search import BeamState, beam_step

        beams = BeamState(scores=state["scores"], pool_scores=state["pool_scores"],
                          pool_rows=state["pool_rows"], pool_steps=state["pool_steps"],
                          done=state["done"], step=c["step"])
        tokens, parents, new, _status = beam_step(
            state["logits"], beams, eos_token_id=state["eos"], pad_token_id=PAD,
            length_penalty=c["penalty"], early_stopping=c["early"], allow_mask=state["mask"])
        return (tokens, parents, new.scores, new.pool_scores, new.pool_rows, new.pool_steps,
                new.done)
    if c["kind"] == "reorder":
        from graspo_amd.beam_search import reorder_states_

        # the step's own parents: no look at them is waited for
        reorder_states_(state["states"], state["parents"], c["beams"], check_status=False)
        return state["cache"]
    if c["kind"] == "expand":
        from graspo_amd.beam_search import expand_states

        return expand_states(state["states"], c["beams"])
    from graspo_amd.lora import lora_add

    # a decode loop's and a trainer's adapter numbers are its own
    out = lora_add(state["base"], state["x"], state["a"], state["b"], adapter_ids=state["ids"],
                   scaling=state["scaling"], check_status=False)
    if not c["grad"]:
        return out
    return out.detach(), *torch.autograd.grad(out, [state["x"], state["a"], state["b"]],
                                              state["g"])


def _plain_beam(state):
    c = state["case"]
    G, K, V = c["groups"], c["beams"], c["vocab"]
    n, inf = 2 * K, float("inf")
    x = state["logits"].double()
    top = x.amax(1, keepdim=True)
    x.sub_(top)
    lse = x.exp().sum(1, keepdim=True).log_()
    x.sub_(lse).add_(state["scores"].reshape(-1, 1))
    if state["mask"] is not None:
        at = torch.arange(V, device="cuda")
        x[(state["mask"][:, at // 32] >> (at % 32)) & 1 == 0] = -inf
    # equal scores keep the order of beams and tokens
    score, flat = x.view(G, K * V).sort(dim=1, descending=True, stable=True)
    score, flat = score[:, :n].clone(), flat[:, :n].clone()
    del x
    beam, token, score = flat // V, flat % V, score.float()
    t1 = (c["step"] + 1.0) ** c["penalty"]
    ended = token == state["eos"]
    # finished candidates among the first K join the pool
    fresh = torch.where(ended[:, :K], (score[:, :K].double() / t1).float(), -inf)
    first = torch.arange(G, device="cuda").unsqueeze(1) * K
    pool = torch.cat([state["pool_scores"], fresh], 1)
    rows = torch.cat([state["pool_rows"], (first + beam[:, :K]).int()], 1)
    steps = torch.cat([state["pool_steps"], torch.full_like(state["pool_steps"], c["step"])], 1)
    pool, at = pool.sort(dim=1, descending=True, stable=True)
    pool, at = pool[:, :K], at[:, :K]
    empty = pool == -inf
    rows = rows.gather(1, at).masked_fill(empty, -1)
    steps = steps.gather(1, at).masked_fill(empty, -1)
    # the first K others go on; a beam's best one stays in its slot
    _, go = ended.int().sort(dim=1, stable=True)
    go = go[:, :K]
    beam, token, score = beam.gather(1, go), token.gather(1, go), score.gather(1, go)
    earlier = torch.ones((K, K), device="cuda").tril(-1).bool()
    again = ((beam.unsqueeze(2) == beam.unsqueeze(1)) & earlier).any(2)
    slots = torch.arange(K, device="cuda")
    taken = (slots.view(1, K, 1) == beam.unsqueeze(1)).any(2)
    free = taken.int().sort(dim=1, stable=True).indices
    slot = torch.where(again, free.gather(1, (again.cumsum(1) - 1).clamp(min=0)), beam)
    tokens = torch.empty_like(token).scatter_(1, slot, token)
    parents = torch.empty_like(beam).scatter_(1, slot, beam)
    scores = torch.empty_like(score).scatter_(1, slot, score)
    full = pool[:, -1] > -inf
    if not c["early"]:
        full = full & (pool[:, -1] >= (scores.amax(1).double() / t1).float())
    # groups that were done stay as they are
    old = state["done"].unsqueeze(1)
    tokens = torch.where(old, PAD, tokens).reshape(-1)
    parents = (torch.where(old, slots, parents) + first).int().reshape(-1)
    return (tokens, parents, torch.where(old, state["scores"], scores),
            torch.where(old, state["pool_scores"], pool),
            torch.where(old, state["pool_rows"], rows),
            torch.where(old, state["pool_steps"], steps), state["done"] | full)


@torch.no_grad()
def _plain(state):
    c = state["case"]
    if c["kind"] == "beam":
        return _plain_beam(state)
    if c["kind"] == "reorder":
        state["live"].copy_(state["live"].index_select(1, state["parents"].long()))
        return state["cache"]
    if c["kind"] == "expand":
        return list(state["live"].repeat_interleave(c["beams"], dim=1).unbind(0))
    ids = state["ids"].long()
    at = ids.clamp(min=0)
    s = torch.where(ids >= 0, state["scaling"][at], 0.0).view(-1, 1, 1)
    x = state["x"].float()
    a = state["a"].float()[at]
    b = state["b"].float()[at]
    u = torch.matmul(x, a.transpose(1, 2).contiguous()) * s
    out = state["base"] + torch.matmul(u, b.transpose(1, 2).contiguous())
    out = out.to(state["base"].dtype)
    if not c["grad"]:
        return out
    g = state["g"].float()
    v = torch.matmul(g, b) * s
    gx = torch.matmul(v, a)
    ga = torch.zeros(state["a"].shape, device="cuda")
    ga.index_add_(0, at, torch.matmul(v.transpose(1, 2).contiguous(), x))
    gb = torch.zeros(state["b"].shape, device="cuda")
    gb.index_add_(0, at, torch.matmul(g.transpose(1, 2).contiguous(), u))
    dt = out.dtype
    return out, gx.to(dt), ga.to(dt), gb.to(dt)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------ what it needs

SIZES = {"fp32": 4, "bf16": 2, "fp16": 2, "uint8": 1}


def work(case):
    kind, size = case["kind"], SIZES[case["dtype"]]
    if kind == "beam":
        # dead beams are not read
        rows = case["groups"] * (1 if case["first"] else case["beams"])
        n = rows * case["vocab"]
        # a maximum, an exponential and a sum of each logit
        return {"bytes": n * size + (n // 8 if case["masked"] else 0), "flops": 4 * n}
    if kind in ("reorder", "expand"):
        row = 2 * case["layers"] * case["heads"] * case["length"] * case["dim"] * size
        if kind == "expand":
            return {"bytes": case["groups"] * (1 + case["beams"]) * row, "flops": 0}
        # each replaced row written, and each row that replaces one read once
        kept, dead = case["beams"] - case["dead"], case["dead"]
        read = kept * (1.0 - (1.0 - 1.0 / kept) ** dead)
        # (a step that replaces none reads the parents alone)
        return {"bytes": max(case["groups"] * (dead + read) * row,
                             4 * case["groups"] * case["beams"]), "flops": 0}
    B, S, K, N, r = (case[k] for k in ("batch", "seq", "width", "out", "rank"))
    n = B * S
    live = S * (B - min(case["none"], B - 1))
    e = case["adapters"] * (1.0 - (1.0 - 1.0 / case["adapters"]) ** (live // S))
    weights = e * r * (K + N) * size
    b, f = 2 * n * N * size + live * K * size + weights, 2 * live * r * (K + N)
    if case["grad"]:
        # both inputs once more, x's gradient and the adapters'
        b += live * (N + K) * size + n * K * size + weights
        b += case["adapters"] * r * (K + N) * size
        f *= 3
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------- in 64 bits

def _exact_group(logp, eos, step, t1, early, scores, pool):
    """One group's step by the rules, on the host: `logp` [K, V] in 64 bits
    with the beams' scores added; `pool`: (score, row in the group, step)."""
    K, V = logp.shape
    best, flat = [], logp.reshape(-1).clone()
    for _ in range(2 * K):
        v, i = flat.max(dim=0)
        best.append((v, i))
        flat[i] = -float("inf")
    best = [(float(v), int(i) // V, int(i) % V) for v, i in best]
    pool = list(pool)
    live = []
    for rank, (score, beam, token) in enumerate(best):
        if token == eos:
            if rank < K:
                pool.append((score / t1, beam, step))
        elif len(live) < K:
            live.append((score, beam, token))
    pool = sorted(pool, key=lambda h: -h[0])[:K]
    slots = {}
    for score, beam, token in live:
        slots.setdefault(beam, (score, beam, token))
    rest = list(live)
    for kept in slots.values():
        rest.remove(kept)
    for k in range(K):
        if k not in slots:
            slots[k] = rest.pop(0)
    done = len(pool) == K and (early or pool[-1][0] >= max(s for s, _, _ in live) / t1)
    return [slots[k] for k in range(K)], pool, done


def _exact_beam(case, st):
    G, K, V = case["groups"], case["beams"], case["vocab"]
    t1 = float(case["step"] + 1) ** case["penalty"]
    inf = float("inf")
    tokens, parents, scores, pools, rows, steps, dones = [], [], [], [], [], [], []
    for b in range(G):
        score = st["scores"][b].tolist()
        old = [(s, r - b * K, t) for s, r, t in zip(st["pool_scores"][b].tolist(),
                                                    st["pool_rows"][b].tolist(),
                                                    st["pool_steps"][b].tolist()) if s > -inf]
        done = bool(st["done"][b])
        live = [(s, k, PAD) for k, s in enumerate(score)]
        if not done:
            logp = torch.log_softmax(st["logits"][b * K : (b + 1) * K].to(torch.float64), dim=1)
            logp += st["scores"][b].to(torch.float64).unsqueeze(1)
            if st["mask"] is not None:
                word = st["mask"][b * K : (b + 1) * K].to(torch.int64) & 0xFFFFFFFF
                bit = word.unsqueeze(2).bitwise_right_shift(torch.arange(32, device="cuda")) & 1
                logp.masked_fill_(bit.reshape(K, -1)[:, :V] == 0, -inf)
            live, old, done = _exact_group(logp, st["eos"], case["step"], t1, case["early"], score,
                                           old)
        scores.append([s for s, _, _ in live])
        parents += [b * K + k for _, k, _ in live]
        tokens += [t for _, _, t in live]
        old = old + [(-inf, -1 - b * K, -1)] * (K - len(old))
        pools.append([s for s, _, _ in old])
        rows.append([r + b * K for _, r, _ in old])
        steps.append([t for _, _, t in old])
        dones.append(done)
    i32, f64 = torch.int32, torch.float64
    return (torch.tensor(tokens), torch.tensor(parents, dtype=i32), torch.tensor(scores, dtype=f64),
            torch.tensor(pools, dtype=f64), torch.tensor(rows, dtype=i32),
            torch.tensor(steps, dtype=i32), torch.tensor(dones))


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    if kind == "beam":
        return _exact_beam(case, st)
    if kind == "reorder":
        for t in st["states"]:
            old = t.clone()
            for row, parent in enumerate(st["parents"].tolist()):
                t[row] = old[parent]
        return st["cache"]
    if kind == "expand":
        return [torch.stack([t] * case["beams"], dim=1).flatten(0, 1) for t in st["states"]]
    out = st["base"].to(f64)
    x, a, b = (st[k].detach().to(f64) for k in ("x", "a", "b"))
    gx, ga, gb = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    g = st["g"].to(f64) if case["grad"] else None
    for e in range(case["adapters"]):
        seqs = torch.nonzero(st["ids"] == e).flatten()
        if not seqs.numel():
            continue
        s = float(st["scaling"][e])
        rows = x[seqs].flatten(0, 1)
        low = rows @ a[e].t()
        out[seqs] += (s * (low @ b[e].t())).view(len(seqs), case["seq"], -1)
        if case["grad"]:
            grows = s * g[seqs].flatten(0, 1)
            back = grows @ b[e]
            gx[seqs] = (back @ a[e]).view(len(seqs), case["seq"], -1)
            ga[e] = back.t() @ rows
            gb[e] = grows.t() @ low
    return (out, gx, ga, gb) if case["grad"] else out
