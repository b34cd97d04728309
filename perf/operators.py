"""The operators at the vocabulary ends of a sequence model, as cases to time
and compare: log-probabilities of given tokens (with entropy, top alternatives
and their reverse), distillation from a teacher's top logits (loss, and loss
with gradient) and the scaled embedding lookup (forward, and with the table's
gradient).

``run`` computes the plain form, elementary torch operations in 32 bits (64
where long sums need it), or, where ``own`` is true, makes the calls a user
makes of ``dabsn_b200``.  ``exact`` gives the same values from the definitions
in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _score(name, rows, vocab, dtype, *, top_k=0, train=False, temperature=1.0, ignored=0.0,
           masked="none", pad=0):
    return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "dtype": dtype,
            "top_k": top_k, "train": train, "temperature": temperature, "ignored": ignored,
            "masked": masked, "pad": pad}


def _distill(name, rows, vocab, dtype, entries, *, train, temperature=1.0, ignored=0.0, pad=0,
             reduction="mean"):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype,
            "entries": entries, "train": train, "temperature": temperature, "ignored": ignored,
            "pad": pad, "reduction": reduction}


def _embed(name, tokens, vocab, width, dtype, out, *, train, scale=1.0, padding=False, zipf=True):
    return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "width": width,
            "dtype": dtype, "out": out, "train": train, "scale": scale, "padding": padding,
            "zipf": zipf}


def listed():
    return [
        # the next tokens of a small batch of requests, with the alternatives a client asks for
        _score("score_next_tokens", 8, 32000, "bf16", top_k=5),
        # policy gradient on the copy task's model: vocabulary 64, 32 sequences of 64 tokens
        _score("score_small_vocab_train", 2048, 64, "fp32", train=True),
        # a teacher's top logits over four sequences of 4096 tokens, to distil from later
        _score("score_corpus_top20", 16384, 32000, "bf16", top_k=20),
        # policy gradient with an entropy bonus over the same, prompts ignored
        _score("score_train", 16384, 32000, "bf16", train=True, ignored=0.1),
        # constrained decoding of a beam: most of an odd-sized vocabulary masked
        _score("score_masked_odd", 333, 32771, "fp32", top_k=64, temperature=0.8,
               masked="grammar"),
        # distilling the small group-theory model: vocabulary 60, 32 sequences of 64 tokens
        _distill("distill_small_vocab", 2048, 60, "fp32", 8, train=True),
        # the loss alone, on a validation batch
        _distill("distill_eval", 4096, 32000, "bf16", 32, train=False, ignored=0.05),
        # a training batch of 16 sequences of 2048 tokens
        _distill("distill_train", 32768, 32000, "bf16", 64, train=True, ignored=0.05),
        # a large odd vocabulary, long lists, a high temperature
        _distill("distill_wide_odd", 515, 128003, "bf16", 128, train=True, temperature=2.0),
        # one token of each of 32 requests, a float table read into bf16
        _embed("embed_next_tokens", 32, 32000, 2048, "fp32", "bf16", train=False, scale=45.25),
        # a training batch of 32 sequences of 4096 tokens at width 2048
        _embed("embed_train", 131072, 32000, 2048, "fp32", "bf16", train=True),
        # a small odd table, with padding
        _embed("embed_train_odd", 4099, 1009, 515, "fp32", "fp32", train=True, scale=0.5,
               padding=True, zipf=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["score", "distill", "embed"])
    train = rng.random() < 0.5
    dtype = rng.choice(["bf16", "fp32"])
    if op == "embed":
        vocab = _log_int(rng, 60, 64000)
        width = _log_int(rng, 64, 4096)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        tokens = _log_int(rng, 1, 131072)
        most = 131072 * 2048  # elements of the largest listed case
        tokens = max(1, min(tokens, most // width))
        vocab = max(60, min(vocab, 32000 * 2048 // width))
        return _embed(None, tokens, vocab, width, dtype, rng.choice(["bf16", "fp32"]), train=train,
                      scale=rng.choice([1.0, 0.5, 45.25]), padding=rng.random() < 0.3,
                      zipf=rng.random() < 0.7)
    vocab = _log_int(rng, 60, 131072)
    if rng.random() < 0.5:
        vocab = max(64, vocab // 64 * 64)
    rows = _log_int(rng, 1, 32768)
    pad = rng.choice([0, 0, 5, 64])
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    ignored = rng.choice([0.0, 0.1, 0.5])
    most = 16384 * 32000 if op == "score" else 32768 * 32000
    rows = max(1, min(rows, most // (BYTES[dtype] // 2) // (vocab + pad)))
    if op == "score":
        masked = rng.choice(["none", "none", "grammar", "lowest"])
        top_k = 0 if train else min(rng.choice([0, 1, 5, 20, 64, 128]), vocab)
        return _score(None, rows, vocab, dtype, top_k=top_k, train=train,
                      temperature=temperature, ignored=ignored, masked=masked, pad=pad)
    entries = min(_log_int(rng, 1, 128), vocab // 2)
    return _distill(None, rows, vocab, dtype, entries, train=train, temperature=temperature,
                    ignored=ignored, pad=pad,
                    reduction=rng.choice(["mean", "sum"]) if train else
                    rng.choice(["mean", "sum", "none"]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _logits(case, gen):
    """Rows of a readout: normal logits around a falling prior over the ids,
    as a view of a wider matrix where the readout is padded."""
    rows, vocab, pad = case["rows"], case["vocab"], case["pad"]
    x = torch.randn(rows, vocab + pad, device="cuda", generator=gen, dtype=TYPES[case["dtype"]])
    prior = -0.5 * torch.log1p(torch.arange(vocab + pad, device="cuda", dtype=torch.float32))
    x.mul_(2.0).add_(prior.to(x.dtype))
    return x[:, :vocab]


def _tokens(case, gen, count):
    """Zipf(1.1) token ids, or uniform ones."""
    vocab = case["vocab"]
    if case.get("zipf", True):
        p = torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64).pow(-1.1)
        edge = torch.cumsum(p, 0) / p.sum()
        u = torch.rand(count, device="cuda", generator=gen, dtype=torch.float64)
        return torch.searchsorted(edge, u).clamp_(max=vocab - 1)
    return torch.randint(0, vocab, (count,), device="cuda", generator=gen)


def _ignored_rows(case, gen):
    """Which rows are padding: a fixed number of them, at random places."""
    rows = case["rows"]
    order = torch.randperm(rows, device="cuda", generator=gen)
    return order[: int(rows * case["ignored"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "embed":
        tokens = _tokens(case, gen, case["tokens"])
        state["padding_idx"] = None
        if case["padding"]:
            state["padding_idx"] = 0
            tokens[torch.rand(case["tokens"], device="cuda", generator=gen) < 0.2] = 0
        state["ids"] = tokens
        state["weight"] = torch.randn(case["vocab"], case["width"], device="cuda", generator=gen,
                                      dtype=TYPES[case["dtype"]])
        if case["train"]:
            state["grad"] = torch.randn(case["tokens"], case["width"], device="cuda",
                                        generator=gen, dtype=TYPES[case["out"]])
        return state
    rows, vocab = case["rows"], case["vocab"]
    x = _logits(case, gen)
    if case["op"] == "score":
        tokens = _tokens(case, gen, rows)
        if case["masked"] != "none":
            # what a grammar leaves: about one id in fifty, in the first rows
            # nothing, one or a few (the given token is always among them
            # where any is)
            low = -math.inf if case["masked"] == "grammar" else torch.finfo(x.dtype).min
            keep = torch.rand(rows, vocab, device="cuda", generator=gen) < 0.02
            keep[: min(4, rows)] = False
            if rows > 2:
                keep[2:4, : 7] = True
            keep.scatter_(1, tokens[:, None], True)
            if rows > 4:
                keep[0] = False
            x = x.masked_fill_(~keep, low)
        tokens[_ignored_rows(case, gen)] = IGNORE
        state["tokens"] = tokens
        if case["train"]:
            state["grad_log_prob"] = torch.randn(rows, device="cuda", generator=gen) / rows
            state["grad_entropy"] = torch.full((rows,), 0.01 / rows, device="cuda")
    else:
        # the teacher's lists: distinct ids that lean to the frequent ones,
        # falling logits, shorter lists in some rows
        k = case["entries"]
        first = _tokens(case, gen, rows)
        stride = 1 + vocab // (2 * k)
        ids = (first[:, None] + torch.arange(k, device="cuda") * stride) % vocab
        logits = torch.randn(rows, k, device="cuda", generator=gen) * 2.0
        logits = torch.sort(logits, dim=-1, descending=True).values
        lift = (logits + 8.0).to(x.dtype)
        x.scatter_add_(1, ids, lift)  # a student that has learnt some of it
        length = torch.randint(max(1, k // 2), k + 1, (rows,), device="cuda", generator=gen)
        ids = torch.where(torch.arange(k, device="cuda") < length[:, None], ids, IGNORE)
        ids[_ignored_rows(case, gen)] = IGNORE
        state["teacher_tokens"], state["teacher_logits"] = ids, logits
    state["logits"] = x
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    if state["op"] == "score":
        return _plain_score(state)
    if state["op"] == "distill":
        return _plain_distill(state)
    return _plain_embed(state)


def _own(state):
    import dabsn_b200

    if state["op"] == "score":
        x = state["logits"]
        if state["train"]:
            x = x.detach().requires_grad_()
        out = dabsn_b200.token_log_probs(x, state["tokens"], top_k=state["top_k"],
                                         temperature=state["temperature"], ignore_index=IGNORE)
        if state["train"]:
            (dx,) = torch.autograd.grad((out.log_prob, out.entropy), x,
                                        (state["grad_log_prob"], state["grad_entropy"]))
            return {"log_prob": out.log_prob, "entropy": out.entropy, "dlogits": dx}
        result = {"log_prob": out.log_prob, "entropy": out.entropy}
        if state["top_k"]:
            result |= {"top_log_probs": out.top_log_probs, "top_tokens": out.top_tokens}
        return result
    if state["op"] == "distill":
        x = state["logits"]
        if state["train"]:
            x = x.detach().requires_grad_()
        loss = dabsn_b200.distillation_loss(
            x, state["teacher_tokens"], state["teacher_logits"],
            temperature=state["temperature"], ignore_index=IGNORE, reduction=state["reduction"])
        if state["train"]:
            (dx,) = torch.autograd.grad(loss, x)
            return {"loss": loss.detach(), "dlogits": dx}
        return {"loss": loss}
    weight = state["weight"]
    if state["train"]:
        weight = weight.detach().requires_grad_()
    out = dabsn_b200.embedding(state["ids"], weight, scale=state["scale"],
                               padding_idx=state["padding_idx"], dtype=TYPES[state["out"]])
    if state["train"]:
        (dw,) = torch.autograd.grad(out, weight, state["grad"])
        return {"out": out.detach(), "dweight": dw}
    return {"out": out}


def _softmax_parts(x, temperature):
    """(d, e, s): (x - max) / T, its exponential and the row's sum; a row of
    nothing but -inf has s = 0."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = (x - m) / temperature
    e = torch.exp(d)
    return d, e, e.sum(-1, keepdim=True)


def _plain_score(state):
    x = state["logits"].float()
    tokens, T, k = state["tokens"], state["temperature"], state["top_k"]
    valid = tokens != IGNORE
    d, e, s = _softmax_parts(x, T)
    empty = s == 0
    s = torch.where(empty, torch.ones_like(s), s)
    log_s = torch.log(s)
    p = e / s
    finite = torch.where(e > 0, d, torch.zeros_like(d))
    entropy = (log_s - (p * finite).sum(-1, keepdim=True)).squeeze(-1)
    at = tokens.clamp(min=0)[:, None]
    log_prob = (d.gather(1, at) - log_s).squeeze(-1)
    log_prob = torch.where(empty.squeeze(-1), -math.inf, log_prob)
    log_prob = torch.where(valid, log_prob, 0.0)
    entropy = torch.where(valid & ~empty.squeeze(-1), entropy, 0.0)
    result = {"log_prob": log_prob, "entropy": entropy}
    if state["train"]:
        g = torch.where(valid, state["grad_log_prob"], 0.0)[:, None]
        h = torch.where(valid, state["grad_entropy"], 0.0)[:, None]
        dx = -p * (g + h * (finite - log_s + entropy[:, None]))
        hit = g * ~empty
        dx.scatter_add_(1, at, hit)
        return result | {"dlogits": (dx / T).to(state["logits"].dtype)}
    if k:
        top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        ids = ids[:, :k]
        top = d.gather(1, ids) - log_s
        top = torch.where(empty | ~valid[:, None], -math.inf, top)
        result |= {"top_log_probs": top, "top_tokens": torch.where(valid[:, None], ids, -1)}
    return result


def _plain_distill(state):
    x = state["logits"].float()
    ids, T = state["teacher_tokens"], state["temperature"]
    here = ids != IGNORE
    t = torch.where(here, state["teacher_logits"].float() / T, -math.inf)
    m = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(m == -math.inf, torch.zeros_like(m), m))
    sum_e = e.sum(-1, keepdim=True)
    valid = sum_e.squeeze(-1) > 0
    q = e / torch.where(sum_e > 0, sum_e, torch.ones_like(sum_e))
    d, e, s = _softmax_parts(x, T)
    log_s = torch.log(s)
    at = ids.clamp(min=0)
    log_p = d.gather(1, at) - log_s
    log_q = torch.log(torch.where(q > 0, q, torch.ones_like(q)))
    row = T * T * torch.where(q > 0, q * (log_q - log_p), torch.zeros_like(q)).sum(-1)
    if state["reduction"] == "none":
        return {"loss": row}
    # a long sum of rows, and the number they are divided by
    loss = row.double().sum()
    count = valid.sum().clamp(min=1) if state["reduction"] == "mean" else 1
    result = {"loss": (loss / count).float()}
    if state["train"]:
        dx = e / s * valid[:, None]
        dx.scatter_add_(1, at, -q)
        result["dlogits"] = (dx * (T / count)).to(state["logits"].dtype)
    return result


def _plain_embed(state):
    weight, ids, scale = state["weight"], state["ids"], state["scale"]
    out = (weight[ids].float() * scale).to(TYPES[state["out"]])
    if not state["train"]:
        return {"out": out}
    g = state["grad"].double()  # long sums: the most frequent token has thousands of rows
    if state["padding_idx"] is not None:
        g = g * (ids != state["padding_idx"])[:, None]
    dw = torch.zeros(weight.shape, device=weight.device, dtype=torch.float64)
    dw.index_add_(0, ids, g)
    return {"out": out, "dweight": (dw * scale).to(weight.dtype)}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _rows_used(case):
    """Expected number of table rows that the tokens read."""
    vocab, count = case["vocab"], case["tokens"]
    if not case["zipf"]:
        return vocab * -math.expm1(count * math.log1p(-1.0 / vocab)) if vocab > 1 else 1.0
    total = sum(k ** -1.1 for k in range(1, vocab + 1))
    return sum(-math.expm1(count * math.log1p(-min(k ** -1.1 / total, 1 - 1e-12)))
               for k in range(1, vocab + 1))


def work(case):
    if case["op"] == "embed":
        n, width = case["tokens"], case["width"]
        out = n * width * BYTES[case["out"]]
        bytes_ = 8 * n + _rows_used(case) * width * BYTES[case["dtype"]] + out
        flops = n * width
        if case["train"]:
            bytes_ += out + case["vocab"] * width * BYTES[case["dtype"]]
            flops += n * width
        return {"bytes": bytes_, "flops": flops}
    rows, vocab, size = case["rows"], case["vocab"], BYTES[case["dtype"]]
    live = rows - int(rows * case["ignored"])
    bytes_ = live * vocab * size  # padding rows need not be read
    flops = 4 * live * vocab
    if case["op"] == "score":
        bytes_ += rows * (8 + 8 + 12 * case["top_k"])
        flops += 2 * live * vocab
        if case["train"]:
            bytes_ += rows * 8
            flops += 4 * live * vocab
    else:
        bytes_ += rows * case["entries"] * 12
        flops += 2 * live * vocab if case["train"] else 0
    if case["train"]:
        bytes_ += rows * vocab * size
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embed":
        return _exact_embed(state)
    logp = torch.log_softmax(state["logits"].double() / state["temperature"], dim=-1)
    if case["op"] == "score":
        return _exact_score(state, logp)
    return _exact_distill(state, logp)


def _exact_score(state, logp):
    # log_softmax of a row of nothing but -inf is NaN throughout
    empty = logp[:, 0].isnan()
    live = state["tokens"] != IGNORE
    pick = torch.arange(len(empty), device=logp.device)
    log_prob = logp[pick, torch.where(live, state["tokens"], 0)]
    log_prob[empty] = -math.inf
    log_prob[~live] = 0
    entropy = torch.special.entr(torch.exp(logp)).sum(-1)
    # entr() of a probability that underflows loses nothing that 64 bits hold
    entropy[empty | ~live] = 0
    result = {"log_prob": log_prob, "entropy": entropy}
    if state["train"]:
        p = torch.exp(logp)
        surprise = torch.where(p > 0, logp, 0.0) + entropy[:, None]
        dx = p * surprise * -state["grad_entropy"].double()[:, None]
        dx -= p * state["grad_log_prob"].double()[:, None]
        dx[pick[live], state["tokens"][live]] += state["grad_log_prob"].double()[live]
        dx[empty | ~live] = 0
        return result | {"dlogits": dx / state["temperature"]}
    if state["top_k"]:
        logp[empty | ~live] = -math.inf
        result |= {"top_log_probs": torch.topk(logp, state["top_k"], dim=-1).values,
                   "top_tokens": None}
    return result


def _exact_distill(state, logp):
    T = state["temperature"]
    ids = state["teacher_tokens"]
    teacher = state["teacher_logits"].double() / T
    log_q = torch.log_softmax(teacher.masked_fill(ids == IGNORE, -math.inf), dim=-1)
    valid = ~log_q[:, 0].isnan()
    q = torch.where(valid[:, None], torch.exp(log_q), 0.0)
    entry = torch.where(q > 0, q * (log_q - logp.gather(1, ids.clamp(min=0))), 0.0)
    row = T ** 2 * entry.sum(-1)
    if state["reduction"] == "none":
        return {"loss": row}
    share = 1.0 / max(1, int(valid.sum())) if state["reduction"] == "mean" else 1.0
    result = {"loss": row.sum() * share}
    if state["train"]:
        dx = logp.exp_()
        dx[~valid] = 0
        rows = torch.arange(len(ids), device=ids.device)[:, None].expand_as(ids)
        dx.index_put_((rows, ids.clamp(min=0)), -q, accumulate=True)
        result["dlogits"] = dx.mul_(T * share)
    return result


def _exact_embed(state):
    ids, scale = state["ids"], state["scale"]
    out = state["weight"].double().index_select(0, ids) * scale
    if not state["train"]:
        return {"out": out}
    # sums over runs of equal tokens, as differences of running sums
    order = torch.argsort(ids, stable=True)
    g = state["grad"].double()[order]
    keys = ids[order]
    if state["padding_idx"] is not None:
        g[keys == state["padding_idx"]] = 0
    edge = torch.cat((torch.zeros_like(g[:1]), torch.cumsum(g, 0)))
    bound = torch.searchsorted(keys, torch.arange(state["vocab"] + 1, device=ids.device))
    sums = edge[bound[1:]] - edge[bound[:-1]]
    return {"out": out, "dweight": sums * scale}
