"""The operators at a language model's two vocabulary ends, measured as a user calls them.

  embed     the scaled token embedding; in training with the gradient of its table, each
            table row the sum of its tokens' gradient rows in token order
  logprobs  log probabilities of given tokens with the rows' entropy and top alternatives;
            in training with the gradient of the logits. ``linear`` starts from the hidden
            rows and the readout's weight and bias instead of from logits
  distill   distillation from a teacher's top logits, loss and gradient. ``rest`` counts the
            probability that the teacher leaves to the tokens not listed; ``linear`` as above

A case of ``logprobs`` or ``distill`` has ``rows`` tokens of a vocabulary of ``vocab`` words.
With ``own`` the calls are the package's, else the same formulas in elementary operations in
32 bits. ``exact`` evaluates the definitions in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # Streaming decode of one sequence: the sampled token's log probability and the five
        # likeliest alternatives a client asks for. Latency is all there is.
        dict(name="logprobs_one", kind="logprobs", dtype="bf16", rows=1, vocab=32000, top=5,
             temperature=1.0, masked=False, train=False),
        # One step of the streaming decode benchmark's batch of 256.
        dict(name="logprobs_batch", kind="logprobs", dtype="bf16", rows=256, vocab=32000, top=20,
             temperature=0.8, masked=True, train=False),
        # A teacher's top 64 over a scored text, fp32 logits of an odd vocabulary.
        dict(name="logprobs_top", kind="logprobs", dtype="fp32", rows=4099, vocab=50021, top=64,
             temperature=1.0, masked=False, train=False),
        # Policy-gradient step: log probabilities with an entropy bonus, forward and backward.
        dict(name="logprobs_train", kind="logprobs", dtype="bf16", rows=8192, vocab=32000, top=0,
             temperature=1.0, masked=False, train=True),
        # Scoring a text from the hidden rows of the streaming model's readout.
        dict(name="logprobs_linear", kind="logprobs_linear", dtype="bf16", rows=4096, width=2048,
             vocab=32000, temperature=1.0),
        # The synthetic copy workload's training shape: 32 x 64 tokens of 65 words.
        dict(name="distill_copy", kind="distill", dtype="fp32", rows=2048, vocab=65, top=8,
             temperature=1.0, rest=False),
        # A readout of 32,000 words, teacher's top 64 and the rest, softened.
        dict(name="distill_wide", kind="distill", dtype="bf16", rows=8192, vocab=32000, top=64,
             temperature=2.0, rest=True),
        # fp32 logits of an odd vocabulary: rows that start at odd addresses.
        dict(name="distill_odd", kind="distill", dtype="fp32", rows=3001, vocab=50021, top=37,
             temperature=1.0, rest=False),
        # The readout and its distillation without logits in memory, with all three gradients.
        dict(name="distill_linear", kind="distill_linear", dtype="bf16", rows=8192, width=2048,
             vocab=32000, top=32, temperature=1.0, rest=True),
        # The token lookup of a decode step of 256 sequences.
        dict(name="embed_decode", kind="embed", dtype="bf16", tokens=256, vocab=32000, width=2048,
             train=False),
        # The group-tracking model (60 words, width 512) over batches of 16 x 4096 tokens: each
        # word the sum of a thousand rows and more.
        dict(name="embed_groups", kind="embed", dtype="fp32", tokens=65536, vocab=60, width=512,
             train=True),
        # The wide single-layer model's step: 16 x 4096 tokens of 32,000 words, width 4096.
        dict(name="embed_wide", kind="embed", dtype="bf16", tokens=65536, vocab=32000, width=4096,
             train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("logprobs", "logprobs", "logprobs_linear", "distill", "distill",
                       "distill_linear", "embed", "embed"))
    dtype = rng.choice(("fp32", "bf16"))
    temperature = rng.choice((0.7, 1.0, 2.0))
    if kind == "embed":
        width = _log(rng, 24, 4096)
        vocab = _log(rng, 60, 65000)
        train = rng.random() < 0.7
        # as much as the widest listed step moves
        tokens = _log(rng, 1, min(200000, 260_000_000 // width))
        return dict(kind=kind, dtype=dtype, tokens=tokens, vocab=vocab, width=width, train=train)
    if kind.endswith("_linear"):
        width, vocab = _log(rng, 64, 2048), _log(rng, 64, 50000)
        rows = _log(rng, 64, min(16384, 120_000_000_000 // (width * vocab)))
        # fp32 readouts run their products in fp32 on both sides: a fraction of the rows
        rows = max(64, rows // 8) if dtype == "fp32" else rows
        case = dict(kind=kind, dtype=dtype, rows=rows, width=width, vocab=vocab,
                    temperature=temperature)
        if kind == "distill_linear":
            case.update(top=min(vocab, rng.randint(1, 100)), rest=rng.random() < 0.5)
        return case
    vocab = _log(rng, 60, 150000)
    rows = _log(rng, 1, min(20000, 150_000_000 // vocab))
    if kind == "logprobs":
        return dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab,
                    top=rng.choice((0, 1, min(vocab, rng.randint(2, 128)))),
                    temperature=temperature, masked=rng.random() < 0.5, train=rng.random() < 0.4)
    return dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab, top=min(vocab, rng.randint(1, 100)),
                temperature=temperature, rest=rng.random() < 0.5)


def _teacher(g, student, case):
    """What a teacher's scoring pass leaves: its top logits and their tokens a row (fewer for
    some rows, none for the padding at the end), and the log of its normaliser."""
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    logits = torch.randn(rows, vocab, generator=g, device=DEVICE).mul_(1.5).add_(student.float())
    values, tokens = logits.topk(top, dim=1)
    lse = torch.logsumexp(logits / case["temperature"], dim=1)
    short = torch.rand(rows, generator=g, device=DEVICE) < 0.05
    tokens[:, top // 2 + 1:].masked_fill_(short[:, None], IGNORE)
    tokens[rows - rows // 50:] = IGNORE
    return values, tokens, lse if case["rest"] else None


def _student(g, rows, vocab):
    """Logits of a trained model: a spread of 2.5, and one likely token a row."""
    x = torch.randn(rows, vocab, generator=g, device=DEVICE).mul_(2.5)
    likely = torch.randint(0, vocab, (rows, 1), generator=g, device=DEVICE)
    return x.scatter_add_(1, likely, torch.rand(rows, 1, generator=g, device=DEVICE) * 12), likely


def _readout(g, case, dtype):
    h = torch.randn(case["rows"], case["width"], generator=g, device=DEVICE).to(dtype)
    w = torch.randn(case["vocab"], case["width"], generator=g, device=DEVICE)
    w = w.mul_(2.5 / math.sqrt(case["width"])).to(dtype)
    b = torch.randn(case["vocab"], generator=g, device=DEVICE).mul_(0.5).to(dtype)
    return h, w, b


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, kind = TYPES[case["dtype"]], case["kind"]
    state = dict(case=case, kind=kind)
    if kind == "embed":
        vocab, width, tokens = case["vocab"], case["width"], case["tokens"]
        weight = torch.randn(vocab, width, generator=g, device=DEVICE).mul_(0.02).to(dtype)
        # Word frequencies fall as one over the rank, as in a text.
        share = 1.0 / (torch.arange(vocab, device=DEVICE, dtype=torch.float32) + 2.7)
        ids = torch.multinomial(share, tokens, replacement=True, generator=g)
        state.update(weight=weight, ids=ids, scale=math.sqrt(width))
        if case["train"]:
            state["grad"] = torch.randn(tokens, width, generator=g, device=DEVICE).to(dtype)
            state["weight"].requires_grad_(True)
        return state
    rows, vocab = case["rows"], case["vocab"]
    if kind.endswith("_linear"):
        h, w, b = _readout(g, case, dtype)
        state.update(hidden=h, weight=w, bias=b)
        if kind == "logprobs_linear":
            state["targets"] = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
            state["targets"][rows - rows // 50:] = IGNORE
        else:
            logits = torch.addmm(b, h, w.t())
            state["values"], state["tokens"], state["lse"] = _teacher(g, logits, case)
            for x in (h, w, b):
                x.requires_grad_(True)
        return state
    x, likely = _student(g, rows, vocab)
    if kind == "logprobs":
        # Half of the given tokens are the likely ones; a constrained row rules words out.
        other = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
        pick = torch.rand(rows, generator=g, device=DEVICE) < 0.5
        state["targets"] = torch.where(pick, likely[:, 0], other)
        if case["masked"]:
            keep = torch.rand(rows, vocab, generator=g, device=DEVICE) < 0.3
            x.masked_fill_(~keep.scatter_(1, state["targets"][:, None], True), -math.inf)
        state["logits"] = x.to(dtype)
        if case["train"]:
            state["logits"].requires_grad_(True)
            state["g_logprob"] = torch.randn(rows, generator=g, device=DEVICE)
            state["g_entropy"] = torch.full((rows,), 0.01, device=DEVICE)
        return state
    state["logits"] = x.to(dtype)
    state["values"], state["tokens"], state["lse"] = _teacher(g, state["logits"], case)
    state["logits"].requires_grad_(True)
    return state


# ---- the formulas in elementary operations, 32 bits ------------------------------------------
def _plain_logprobs(x, targets, case):
    z = x.float() / case["temperature"]
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(dim=1, keepdim=True)
    lse = m + torch.log(s)
    p = e / s
    logp = z - lse
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(dim=1)
    valid = targets != IGNORE
    at = targets.clamp(min=0)[:, None]
    logprob = torch.where(valid, logp.gather(1, at)[:, 0], 0.0)
    return z, logp, p, logprob, entropy, valid, at


def _plain_logprobs_grad(logp, p, entropy, valid, at, case, g_logprob, g_entropy, dtype):
    g = torch.where(valid, g_logprob, 0.0)[:, None]
    d = -p * g - torch.where(p > 0, p * (logp + entropy[:, None]), 0.0) * g_entropy[:, None]
    d.scatter_add_(1, at, g)
    return (d / case["temperature"]).to(dtype)


def _plain_distill(x, values, tokens, lse, case):
    """(loss, gradient of the logits, 32 bits); the teacher's few weights in 64 bits, where
    one minus their sum would lose what is left."""
    t = case["temperature"]
    z = x.float() / t
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(dim=1, keepdim=True)
    here = tokens != IGNORE
    at = tokens.clamp(min=0)
    u = torch.where(here, values.double() / t, -math.inf)
    some = here.any(dim=1)
    if lse is None:
        top = torch.where(some[:, None], u.amax(dim=1, keepdim=True), 0.0)
        w = torch.exp(u - top)
        total = w.sum(dim=1, keepdim=True).clamp_min(1e-300)
        q, logq = w / total, u - top - torch.log(total)
    else:
        logq = u - lse.double()[:, None]
        q = torch.exp(logq)
    logp = z.gather(1, at) - (m + torch.log(s))
    rows = torch.where(q > 0, q * (logq - logp.double()), 0.0).sum(dim=1)
    q32 = q.float()
    if lse is None:
        d = e * (q32.sum(dim=1, keepdim=True) / s)
    else:
        # Words whose place holds a listed token leave the rest's sum.
        hits = torch.zeros_like(e).scatter_add_(1, at, here.float())
        listed_ = hits > 0
        left = torch.where(listed_, 0.0, e).sum(dim=1)
        rest = (1 - q.sum(dim=1)).clamp_min(0.0)
        live = (rest > 0) & (left > 0)
        term = rest * (torch.log(rest) - torch.log(left.double()) + torch.log(s[:, 0].double()))
        rows = rows + torch.where(live, term, 0.0)
        rest32 = torch.where(live, rest, 0.0).float()
        total = q32.sum(dim=1) + rest32
        d = e * (total[:, None] / s)
        back = torch.where(live, rest32 / left, 0.0)[:, None]
        d = d - torch.where(listed_, 0.0, e * back)
    d.scatter_add_(1, at, torch.where(here, -q32, 0.0))
    count = some.sum().clamp_min(1)
    d = d * (some[:, None] * (t / count))
    loss = t * t * torch.where(some, rows, 0.0).sum() / count
    return loss.float(), d


def _plain(state):
    kind, case = state["kind"], state["case"]
    if kind == "embed":
        ids, w, scale = state["ids"], state["weight"].detach(), state["scale"]
        out = (w.float()[ids] * scale).to(w.dtype)
        if not case["train"]:
            return {"out": out}
        d = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
        d.index_add_(0, ids, state["grad"].float())
        return {"out": out, "grad": (d * scale).to(w.dtype)}
    if kind.endswith("_linear"):
        h, w, b = (state[k].detach().float() for k in ("hidden", "weight", "bias"))
        x = torch.addmm(b, h, w.t())
    else:
        x = state["logits"].detach()
    if kind.startswith("logprobs"):
        z, logp, p, logprob, entropy, valid, at = _plain_logprobs(x, state["targets"], case)
        out = {"logprob": logprob, "entropy": entropy}
        if case.get("top"):
            best, index = x.float().sort(dim=1, descending=True, stable=True)
            index = index[:, :case["top"]].contiguous()
            out.update(top=logp.gather(1, index), tokens=index)
        if case.get("train"):
            out["grad"] = _plain_logprobs_grad(logp, p, entropy, valid, at, case,
                                               state["g_logprob"], state["g_entropy"], x.dtype)
        return out
    loss, d = _plain_distill(x, state["values"], state["tokens"], state["lse"], case)
    if kind == "distill":
        return {"loss": loss, "grad": d.to(x.dtype)}
    t = state["hidden"].dtype
    return {"loss": loss, "hidden": (d @ w).to(t), "weight": (d.t() @ h).to(t),
            "bias": d.sum(dim=0).to(t)}


# ---- the package's calls ---------------------------------------------------------------------
def _package(state):
    import dabsn_amd

    kind, case = state["kind"], state["case"]
    if kind == "embed":
        out = dabsn_amd.scaled_embedding(state["ids"], state["weight"], scale=state["scale"])
        if not case["train"]:
            return {"out": out}
        (grad,) = torch.autograd.grad(out, state["weight"], state["grad"])
        return {"out": out, "grad": grad}
    if kind == "logprobs_linear":
        r = dabsn_amd.chunked_linear_token_logprobs(
            state["hidden"], state["weight"], state["bias"], state["targets"],
            temperature=case["temperature"], ignore_index=IGNORE)
        return {"logprob": r.logprobs, "entropy": r.entropy}
    if kind == "logprobs":
        r = dabsn_amd.token_logprobs(state["logits"], state["targets"], top=case["top"],
                                     temperature=case["temperature"], ignore_index=IGNORE)
        out = {"logprob": r.logprobs, "entropy": r.entropy}
        if case["top"]:
            out.update(top=r.top_logprobs, tokens=r.top_indices)
        if case["train"]:
            (out["grad"],) = torch.autograd.grad((r.logprobs, r.entropy), state["logits"],
                                                 (state["g_logprob"], state["g_entropy"]))
        return out
    more = dict(temperature=case["temperature"], teacher_lse=state["lse"], ignore_index=IGNORE)
    if kind == "distill":
        loss = dabsn_amd.distillation_from_logits(state["logits"], state["values"],
                                                  state["tokens"], **more)
        (grad,) = torch.autograd.grad(loss, state["logits"])
        return {"loss": loss, "grad": grad}
    leaves = (state["hidden"], state["weight"], state["bias"])
    loss = dabsn_amd.chunked_linear_distillation(*leaves, state["values"], state["tokens"], **more)
    gh, gw, gb = torch.autograd.grad(loss, leaves)
    return {"loss": loss, "hidden": gh, "weight": gw, "bias": gb}


def run(state):
    return _package(state) if own else _plain(state)


def work(case):
    kind, size = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind == "embed":
        n, v, h = case["tokens"], case["vocab"], case["width"]
        rows = min(n, v) * h * size + 8 * n + n * h * size
        return {"bytes": rows + (n * h * size + v * h * size if case["train"] else 0),
                "flops": n * h * (3 if case["train"] else 1)}
    n, v, k = case["rows"], case["vocab"], case.get("top", 0)
    few = n * (12 * k + 24)
    if kind.endswith("_linear"):
        h = case["width"]
        both = 3 if kind == "distill_linear" else 1
        ends = (n * h + v * h + v) * size * (2 if both == 3 else 1)
        return {"bytes": ends + few, "flops": both * 2 * n * v * h + 8 * n * v}
    both = 2 if kind == "distill" or case.get("train") else 1
    return {"bytes": both * n * v * size + few, "flops": both * 6 * n * v}


# ---- the definitions in 64 bits --------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    kind, t = case["kind"], case.get("temperature", 1.0)
    f64 = torch.float64
    if kind == "embed":
        w, scale = state["weight"].detach().to(f64), state["scale"]
        out = {"out": scale * w.index_select(0, state["ids"])}
        if case["train"]:
            total = torch.zeros_like(w).index_add_(0, state["ids"], state["grad"].to(f64))
            out["grad"] = scale * total
        return out
    if kind.endswith("_linear"):
        leaves = [state[k].detach().to(f64) for k in ("hidden", "weight", "bias")]
        x = leaves[0] @ leaves[1].t() + leaves[2]
    else:
        x = state["logits"].detach().to(f64)
    logp = torch.log_softmax(x / t, dim=1)
    p = logp.exp()
    rows = torch.arange(case["rows"], device=DEVICE)
    if kind.startswith("logprobs"):
        known = state["targets"] != IGNORE
        at = torch.where(known, state["targets"], 0)
        entropy = -torch.special.xlogy(p, p).sum(dim=1)
        out = {"logprob": torch.where(known, logp[rows, at], 0.0), "entropy": entropy}
        if case.get("top"):
            out["top"] = logp.topk(case["top"], dim=1).values
            out["tokens"] = None
        if case.get("train"):
            gl, ge = state["g_logprob"].to(f64), state["g_entropy"].to(f64)
            safe = torch.where(p > 0, logp, 0.0)
            grad = -(p * (safe + entropy[:, None])) * ge[:, None]
            grad -= p * (gl * known)[:, None]
            grad[rows, at] += gl * known
            out["grad"] = grad / t
        return out
    present = state["tokens"] != IGNORE
    known = present.any(dim=1)
    count = max(1, int(known.sum()))
    u = torch.where(present, state["values"].to(f64) / t, -math.inf)
    norm = torch.logsumexp(u, dim=1) if state["lse"] is None else state["lse"].to(f64)
    q = torch.where(known[:, None], torch.exp(u - norm[:, None]), 0.0)
    spread = torch.zeros_like(p)  # the teacher's weights over the whole vocabulary
    spread.scatter_add_(1, torch.where(present, state["tokens"], 0), torch.where(present, q, 0.0))
    cross = torch.where(spread > 0, spread * logp, 0.0).sum(dim=1)
    rows_loss = torch.special.xlogy(q, q).sum(dim=1) - cross
    grad = p * spread.sum(dim=1, keepdim=True) - spread
    if state["lse"] is not None:
        taken = torch.zeros_like(p, dtype=torch.int32)
        taken.scatter_add_(1, torch.where(present, state["tokens"], 0), present.to(torch.int32))
        outside = torch.where(taken > 0, 0.0, p)
        left = outside.sum(dim=1)
        rest = (1.0 - q.sum(dim=1)).clamp(min=0.0)
        rest = torch.where(left > 0, rest, 0.0)
        rows_loss += torch.special.xlogy(rest, rest) - torch.special.xlogy(rest, left)
        share = torch.where(left > 0, rest / left, 0.0)
        grad += p * rest[:, None] - outside * share[:, None]
    loss = t * t * (rows_loss * known).sum() / count
    d = grad * (known[:, None] * (t / count))
    if kind == "distill":
        return {"loss": loss, "grad": d}
    return {"loss": loss, "hidden": d @ leaves[1], "weight": d.t() @ leaves[0], "bias": d.sum(dim=0)}
