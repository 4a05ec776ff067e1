"""Two families of operators on the language-model head, as cases that can be timed and compared with their plain forms.

``kind`` says which operator a case is a call of:

  top       from materialised logits: each token's log-probability, rank and entropy and the ``k`` best alternatives with their
            log-probabilities; with ``train`` also the gradient of the logits from gradients on all three
  logits    the head with low-rank adapters of many requests, for the few tokens of a decoding step: logits out
  logprobs  the same head in training: log-probability and entropy of given tokens from hidden states, and the gradients of the
            hidden states and of every adapter (the head itself is frozen)

Sizes: ``tokens``, ``vocab``, ``hidden``; ``adapters`` adapters of rank ``rank``.  ``order`` is how the tokens of a batch belong to
adapters: "runs" (sequences one behind the other, as a packed batch has them), "mixed" (a decoding step: one token per request),
"one" (a single tenant).

With adapter a(t) of token t, scaling s and no adapter where the id is outside [0, adapters):

  z_t = W h_t + s_a B_a (A_a h_t)                           logits, y = z / temperature
  logprob_t = y_t[label] - log sum exp y_t                  0 where the label is outside the vocabulary
  entropy_t = log sum exp y_t - sum softmax(y_t) y_t
  rank_t = 1 + number of columns that sort before the label: larger value first, then the lower column
"""

from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # One decoding step of a few requests that ask for alternatives: launches and latency.
        dict(name="top of a decoding step", kind="top", tokens=8, vocab=151936, k=20, dtype="bf16", temperature=0.7, masked=0.0, train=False),
        # Prompt scoring with alternatives on fp32 logits of a forward pass.
        dict(name="top of prompts", kind="top", tokens=2048, vocab=152064, k=5, dtype="f32", temperature=1.0, masked=0.0, train=False),
        # Constrained decoding of a small vocabulary with added tokens: most of a row is masked, rows start anywhere.
        dict(name="top under a mask", kind="top", tokens=137, vocab=32001, k=8, dtype="bf16", temperature=1.0, masked=0.97, train=False),
        # Distillation on the policy's own alternatives: gradients on the token, the entropy and every alternative.
        dict(name="top in training", kind="top", tokens=4096, vocab=151936, k=32, dtype="bf16", temperature=1.0, masked=0.0, train=True),
        # A single request with its adapter on a small model.
        dict(name="logits of one token", kind="logits", tokens=1, hidden=896, vocab=151936, adapters=4, rank=8, order="one", out="bf16"),
        # A decoding step of requests of several tenants.
        dict(name="logits of a group", kind="logits", tokens=16, hidden=3584, vocab=152064, adapters=8, rank=16, order="mixed", out="bf16"),
        # The same for many tenants, fp32 logits for the sampler.
        dict(name="logits of many tenants", kind="logits", tokens=128, hidden=1536, vocab=151936, adapters=48, rank=32, order="mixed", out="f32"),
        # The last positions of packed prompts: more tokens than a half tile holds, odd sizes.
        dict(name="logits of a ragged batch", kind="logits", tokens=217, hidden=2048, vocab=128261, adapters=5, rank=24, order="runs", out="bf16"),
        # A micro-batch of one sequence of one tenant.
        dict(name="training of one tenant", kind="logprobs", tokens=137, hidden=1536, vocab=151936, adapters=1, rank=16, order="one", temperature=1.0,
             prompt=0.3, entropy_grad=False),
        # Sequences of several tenants in one stream, half of the tokens prompt, an entropy bonus.
        dict(name="training of some tenants", kind="logprobs", tokens=2048, hidden=896, vocab=151936, adapters=6, rank=32, order="runs", temperature=0.7,
             prompt=0.5, entropy_grad=True),
        # Odd sizes, tokens of a dozen tenants.
        dict(name="training on odd sizes", kind="logprobs", tokens=611, hidden=4096, vocab=32001, adapters=12, rank=8, order="runs", temperature=1.0,
             prompt=0.4, entropy_grad=True),
        # A full micro-batch on the headline head.
        dict(name="training of a long batch", kind="logprobs", tokens=8192, hidden=3584, vocab=152064, adapters=4, rank=32, order="runs", temperature=1.0,
             prompt=0.0, entropy_grad=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["top", "logits", "logprobs"])
    vocab = _log(rng, 8000, 152064)
    if kind == "top":
        train = rng.random() < 0.4
        tokens = min(_log(rng, 1, 4096), 4096 * 151936 // vocab)
        masked = rng.choice([0.0, 0.0, 0.9])
        return dict(kind=kind, tokens=tokens, vocab=vocab, k=_log(rng, 1, 64), dtype=rng.choice(["bf16", "f32"]) if tokens <= 2048 else "bf16",
                    temperature=rng.choice([1.0, 0.6, 1.3]), masked=masked, train=train)
    hidden, rank = 64 * _log(rng, 8, 64), 8 * rng.choice([1, 2, 3, 4, 8])
    if kind == "logits":
        adapters = min(_log(rng, 1, 64), 48 * 32 // rank)
        return dict(kind=kind, tokens=_log(rng, 1, 256), hidden=hidden, vocab=vocab, adapters=adapters, rank=rank, order=rng.choice(["runs", "mixed"]),
                    out=rng.choice(["bf16", "f32"]))
    tokens = min(_log(rng, 64, 8192), max(64, 4096 * 3584 * 152064 // (hidden * vocab)))
    return dict(kind=kind, tokens=tokens, hidden=hidden, vocab=vocab, adapters=_log(rng, 1, 12), rank=rank, order=rng.choice(["runs", "runs", "mixed"]),
                temperature=rng.choice([1.0, 0.7]), prompt=rng.choice([0.0, 0.5]), entropy_grad=rng.random() < 0.5)


# -------------------------------------------------------------------------------------------------------------- inputs

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _top_inputs(case, gen):
    T, V, k, dev = case["tokens"], case["vocab"], case["k"], "cuda"
    logits = torch.randn(T, V, generator=gen, device=dev).mul_(2.5)
    # A few tokens of a row stand out, as in a model's output: the label is one of them more often than not.
    peaks = torch.randint(0, V, (T, 4), generator=gen, device=dev)
    logits.scatter_add_(1, peaks, torch.rand(T, 4, generator=gen, device=dev).mul_(12.0))
    labels = torch.where(torch.rand(T, generator=gen, device=dev) < 0.7, peaks[:, 0], torch.randint(0, V, (T,), generator=gen, device=dev))
    if case["masked"]:  # the tokens that a grammar does not allow; the label is allowed
        gone = torch.rand(T, V, generator=gen, device=dev) < case["masked"]
        gone.scatter_(1, labels[:, None], False)
        logits.masked_fill_(gone, -math.inf)
    elif T > 16:  # the first tokens of sequences have no label
        labels[::16] = -100
    state = {"logits": logits.to(_TYPES[case["dtype"]]), "labels": labels}
    if case["train"]:
        state["g"] = torch.randn(T, generator=gen, device=dev)
        state["q"] = torch.randn(T, generator=gen, device=dev).mul_(0.01)
        state["gt"] = torch.rand(T, k, generator=gen, device=dev).mul_(-1.0 / k)
    return state


def _ids(case, gen):
    T, N, dev = case["tokens"], case["adapters"], "cuda"
    if case["order"] == "one":
        return torch.zeros(T, dtype=torch.int64, device=dev)
    if case["order"] == "mixed":  # one token per request; one request in nine has no adapter
        ids = torch.randint(0, N, (T,), generator=gen, device=dev)
        return torch.where(torch.rand(T, generator=gen, device=dev) < 0.11, torch.full_like(ids, -1), ids)
    cuts = torch.sort(torch.randint(0, T + 1, (max(1, 2 * N - 1),), generator=gen, device=dev)).values
    run = torch.bucketize(torch.arange(T, device=dev), cuts, right=True)  # the sequence of a token, 0 .. 2 N - 1
    return torch.randint(0, N, (2 * N,), generator=gen, device=dev)[run]


def _head_inputs(case, gen):
    T, H, V, N, R, dev = case["tokens"], case["hidden"], case["vocab"], case["adapters"], case["rank"], "cuda"
    b16 = torch.bfloat16
    state = {
        "hidden": torch.randn(T, H, generator=gen, device=dev).to(b16),
        "weight": (torch.randn(V, H, generator=gen, device=dev, dtype=b16) * (2.0 / math.sqrt(H))).to(b16),
        "lora_a": (torch.randn(N, R, H, generator=gen, device=dev) * (1.0 / math.sqrt(H))).to(b16),
        "lora_b": (torch.randn(N, V, R, generator=gen, device=dev, dtype=b16) * 0.08).to(b16),
        "scaling": 0.5 + 1.5 * torch.rand(N, generator=gen, device=dev),
        "ids": _ids(case, gen),
    }
    if case["kind"] == "logprobs":
        state["labels"] = torch.randint(0, V, (T,), generator=gen, device=dev)
        graded = (torch.arange(T, device=dev) % max(2, T // 4)) >= int(case["prompt"] * max(2, T // 4))  # four sequences, each with a prompt
        state["g"] = torch.randn(T, generator=gen, device=dev) * graded
        state["q"] = torch.randn(T, generator=gen, device=dev).mul_(0.02) * graded if case["entropy_grad"] else None
        for name in ("hidden", "lora_a", "lora_b"):
            state[name].requires_grad_()
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = _top_inputs(case, gen) if case["kind"] == "top" else _head_inputs(case, gen)
    return {"case": case, **state}


# --------------------------------------------------------------------------------------------------------- plain forms


def _top_plain(s):
    case, logits, labels, k = s["case"], s["logits"], s["labels"], s["case"]["k"]
    T, V = logits.shape
    z = logits.float()
    col = torch.arange(V, device=z.device)
    # One integer per logit that sorts as (value, lower column first): unique, so that ties are settled.
    bits = (z + 0.0).view(torch.int32).to(torch.int64)
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 32) + (V - 1 - col)
    ids = key.topk(k, dim=1).indices
    has = (labels >= 0) & (labels < V)
    safe = torch.where(has, labels, 0)[:, None]
    ranks = torch.where(has, 1 + (key > key.gather(1, safe)).sum(1), 0)
    del key, bits
    rcp = 1.0 / case["temperature"]
    y = z * rcp
    top = y.amax(1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    e = torch.exp(y - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    some = total > 0
    p = torch.where(some, e / total, 0.0)
    spread = torch.where(p > 0, y - top, 0.0)
    mean = (p * spread).sum(1, keepdim=True)
    empty = torch.full_like(lse, -math.inf)
    logprobs = torch.where(has, torch.where(some, y.gather(1, safe) - lse, empty)[:, 0], 0.0)
    out = {
        "logprobs": logprobs,
        "entropy": torch.where(some, torch.log(total) - mean, 0.0)[:, 0],
        "ranks": ranks,
        "top_logprobs": torch.where(some, y.gather(1, ids) - lse, empty),
        "top_ids": ids,
    }
    if case["train"]:
        g = torch.where(has, s["g"], 0.0)[:, None]
        d = p * (-(g + s["gt"].sum(1, keepdim=True)) - s["q"][:, None] * (spread - mean))
        d.scatter_add_(1, safe, g)
        d.scatter_add_(1, ids, s["gt"])
        out["d_logits"] = torch.where(some, d * rcp, 0.0).to(logits.dtype)
    return out


def _selected(s):
    """Which adapter a token has, as a [T, N] matrix of scalings."""
    n = torch.arange(s["lora_a"].shape[0], device=s["ids"].device)
    return (s["ids"][:, None] == n).float() * s["scaling"].float()


def _head_plain(s):
    """Logits in 32 bits, and what the gradients need besides.  All adapters side by side: a token's own one is what its row selects."""
    h, w, a, b = (s[n].detach().float() for n in ("hidden", "weight", "lora_a", "lora_b"))
    N, R, H = a.shape
    chosen = _selected(s).repeat_interleave(R, dim=1)                 # [T, N R]
    a_all, b_all = a.reshape(N * R, H), b.transpose(0, 1).reshape(-1, N * R)
    u = (h @ a_all.T) * chosen
    z = (h @ w.T).addmm_(u, b_all.T)
    return z, h, w, a_all, b_all, u, chosen


def _logits_plain(s):
    return {"logits": _head_plain(s)[0].to(_TYPES[s["case"]["out"]])}


def _logprobs_plain(s):
    case, labels = s["case"], s["labels"]
    N, R, H = s["lora_a"].shape
    rcp = 1.0 / case["temperature"]
    z, h, w, a_all, b_all, u, chosen = _head_plain(s)
    z.mul_(rcp)
    top = z.amax(1, keepdim=True)
    z.sub_(top)
    at_label = z.gather(1, labels[:, None])
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    p = e.div_(total)
    mean = (p * z).sum(1, keepdim=True)
    out = {"logprobs": (at_label - torch.log(total))[:, 0], "entropy": (torch.log(total) - mean)[:, 0]}
    g = s["g"][:, None]
    coef = -g if s["q"] is None else -g - s["q"][:, None] * z.sub_(mean)
    d = p.mul_(coef)
    d.scatter_add_(1, labels[:, None], g)
    d.mul_(rcp)
    du = (d @ b_all) * chosen
    out["d_hidden"] = (d @ w).addmm_(du, a_all).to(torch.bfloat16)
    out["d_lora_a"] = (du.T @ h).reshape(N, R, H).to(torch.bfloat16)
    out["d_lora_b"] = (d.T @ u).reshape(-1, N, R).transpose(0, 1).to(torch.bfloat16)
    return out


# -------------------------------------------------------------------------------------------------- the framework's own


def _top_own(s):
    from skyrl_amd.torch_utils import top_logprobs_from_logits

    case = s["case"]
    if not case["train"]:
        return top_logprobs_from_logits(s["logits"], s["labels"], case["k"], temperature=case["temperature"])._asdict()
    logits = s["logits"].detach().requires_grad_()
    r = top_logprobs_from_logits(logits, s["labels"], case["k"], temperature=case["temperature"])
    (d,) = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), (logits,), (s["g"], s["q"], s["gt"]))
    return {**r._asdict(), "d_logits": d}


def _logits_own(s):
    from skyrl_amd.adapters import adapter_logits

    return {"logits": adapter_logits(s["hidden"], s["weight"], s["lora_a"], s["lora_b"], s["scaling"], s["ids"], dtype=_TYPES[s["case"]["out"]])}


def _logprobs_own(s):
    from skyrl_amd.adapters import adapter_logprobs_from_hidden

    leaves = (s["hidden"], s["lora_a"], s["lora_b"])
    logprobs, entropy = adapter_logprobs_from_hidden(s["hidden"], s["weight"], s["labels"], s["lora_a"], s["lora_b"], s["scaling"], s["ids"],
                                                     temperature=s["case"]["temperature"])
    if s["q"] is None:
        grads = torch.autograd.grad((logprobs,), leaves, (s["g"],))
    else:
        grads = torch.autograd.grad((logprobs, entropy), leaves, (s["g"], s["q"]))
    return {"logprobs": logprobs, "entropy": entropy, "d_hidden": grads[0], "d_lora_a": grads[1], "d_lora_b": grads[2]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return (_top_own if kind == "top" else _logits_own if kind == "logits" else _logprobs_own)(state)
    return (_top_plain if kind == "top" else _logits_plain if kind == "logits" else _logprobs_plain)(state)


# ------------------------------------------------------------------------------------------------------ work and 64 bits


def work(case):
    T, V = case["tokens"], case["vocab"]
    if case["kind"] == "top":
        es = 2 if case["dtype"] == "bf16" else 4
        rows = T * V * es * (2 if case["train"] else 1)
        return {"bytes": rows + T * (24 + 12 * case["k"] + (8 + 4 * case["k"] if case["train"] else 0)), "flops": (12 if case["train"] else 6) * T * V}
    H, N, R = case["hidden"], case["adapters"], case["rank"]
    used = min(N, T)
    operands = 2 * (T * H + V * H + used * R * (H + V))
    if case["kind"] == "logits":
        return {"bytes": operands + T * (8 + V * (2 if case["out"] == "bf16" else 4)), "flops": 2 * T * (V * H + R * (H + V))}
    graded = T - int(case["prompt"] * T)
    return {"bytes": operands + 2 * (T * H + N * R * (H + V)) + 28 * T,
            "flops": 2 * T * (V * H + R * (H + V)) + 2 * graded * (V * H + 2 * R * (H + V))}


def _exact_rows(y, labels, has):
    """Statistics of rows of y (64 bits) by the definition, with the limits of an empty row."""
    top = y.max(dim=1).values
    some = torch.isfinite(top)
    shift = torch.where(some, top, torch.zeros_like(top))
    lse = shift + torch.logsumexp(y - shift[:, None], dim=1)
    p = torch.exp(y - torch.where(some, lse, torch.zeros_like(lse))[:, None])
    logp = torch.where(p > 0, y - lse[:, None], torch.zeros_like(y))
    entropy = -(p * logp).sum(dim=1)
    picked = y[torch.arange(y.shape[0], device=y.device), torch.where(has, labels, torch.zeros_like(labels))]
    logprob = torch.where(some, picked - lse, torch.full_like(lse, -math.inf))
    return torch.where(has, logprob, torch.zeros_like(logprob)), entropy, p, logp, lse, some


def exact(case, seed):
    s = prepare(case, seed)
    T, V, dev = case["tokens"], case["vocab"], s["labels"].device if "labels" in s else s["ids"].device
    block = max(1, (1 << 27) // V)
    parts = []
    if case["kind"] == "top":
        for t in range(0, T, block):
            raw, labels = s["logits"][t:t + block].double(), s["labels"][t:t + block]
            rows = torch.arange(raw.shape[0], device=dev)
            has = (labels >= 0) & (labels < V)
            safe = torch.where(has, labels, torch.zeros_like(labels))
            order = torch.sort(raw, dim=1, descending=True, stable=True).indices
            place = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=dev).expand_as(order))
            ids = order[:, :case["k"]].contiguous()
            y = raw / case["temperature"]
            logprob, entropy, p, logp, lse, some = _exact_rows(y, labels, has)
            tops = torch.where(some[:, None], y.gather(1, ids) - lse[:, None], torch.full_like(ids, -math.inf, dtype=torch.float64))
            part = {"logprobs": logprob, "entropy": entropy, "ranks": torch.where(has, place[rows, safe] + 1, torch.zeros_like(safe)),
                    "top_logprobs": tops, "top_ids": ids}
            if case["train"]:
                g, q, gt = (s[n][t:t + block].double() for n in ("g", "q", "gt"))
                d = -p * (gt.sum(dim=1) + torch.where(has, g, torch.zeros_like(g)))[:, None] - q[:, None] * p * (logp + entropy[:, None])
                d[rows, safe] += torch.where(has, g, torch.zeros_like(g))
                d.scatter_add_(1, ids, gt)
                part["d_logits"] = (d / case["temperature"]).to(torch.float64)
            # 64-bit values of a large gradient are not kept all at once: 32 bits hold them far closer than the type compared.
            parts.append({n: v.float() if n == "d_logits" else v for n, v in part.items()})
        return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}

    h, w = s["hidden"].detach().double(), s["weight"].double()
    a, b = s["lora_a"].detach().double(), s["lora_b"].detach()
    scaling, ids = s["scaling"].double(), s["ids"]
    N, R, H = a.shape
    train = case["kind"] == "logprobs"
    da, db = (torch.zeros_like(a), torch.zeros(N, V, R, dtype=torch.float64, device=dev)) if train else (None, None)
    present = [n for n in range(N) if bool((ids == n).any())]
    for t in range(0, T, block):
        rows = {n: (ids[t:t + block] == n).nonzero()[:, 0] for n in present}
        x = h[t:t + block]
        z = x @ w.T
        for n, at in rows.items():
            if at.numel():
                z[at] += scaling[n] * ((x[at] @ a[n].T) @ b[n].double().T)
        if not train:
            parts.append({"logits": z})
            continue
        labels = s["labels"][t:t + block]
        logprob, entropy, p, logp, _, _ = _exact_rows(z / case["temperature"], labels, torch.ones_like(labels, dtype=torch.bool))
        del z
        g = s["g"][t:t + block].double()
        d = p * -g[:, None]
        if s["q"] is not None:
            d -= s["q"][t:t + block].double()[:, None] * p * (logp + entropy[:, None])
        d[torch.arange(x.shape[0], device=dev), labels] += g
        d /= case["temperature"]
        dx = d @ w
        for n, at in rows.items():
            if at.numel():
                bn = b[n].double()
                dv = scaling[n] * (d[at] @ bn)
                dx[at] += dv @ a[n]
                da[n] += dv.T @ x[at]
                db[n] += d[at].T @ (scaling[n] * (x[at] @ a[n].T))
        parts.append({"logprobs": logprob, "entropy": entropy, "d_hidden": dx})
    out = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    if train:
        out["d_lora_a"], out["d_lora_b"] = da, db
    return out
