"""Operators on rows of logits as timing cases: a teacher's record of its top
logits, the distillation loss on such records with its gradient, and sampling
with temperature, top-k, top-p and min-p from given random numbers.

A case is a dict of plain values. Its "op" is one of
  top      top_logits(logits, k): values, indices, log-mass of the rest
  distill  distillation_loss over a batch of rows; with "train" the logits'
           gradient too (loss.backward()), without it the loss alone
  sample   sample_tokens(logits, uniforms): tokens and their log-probabilities
All carry rows, vocab, "x" (the logits' type) and "pad": columns between the
end of a row and the start of the next (a vocabulary padded for the last
layer's sake, of which only the real part is used).
  top      k, temperature
  distill  k, temperature, "rest" (the record holds the mass outside its top
           logits), "ragged" (lists of different lengths, some rows with none,
           and row weights of which a share is zero)
  sample   temperature, top_k, top_p, min_p; "mixed": every row has parameters
           of its own, as requests served together have

Logits are N(0, 2) with 32 raised positions a row (fewer in small rows), so
that rows run from a sharp answer to a flat one; a student's are near its
teacher's. All of it comes from the seed alone.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
FIXED = 2.0**40  # sampling weights are integers in units of 2^-40 of the row's largest


def _top(rows, vocab, k, *, x="f32", pad=0, temperature=1.0):
    return {"op": "top", "rows": rows, "vocab": vocab, "k": k, "x": x, "pad": pad, "temperature": temperature}


def _distill(rows, vocab, k, *, x="f32", pad=0, temperature=1.0, rest=True, ragged=False, train=True):
    return {"op": "distill", "rows": rows, "vocab": vocab, "k": k, "x": x, "pad": pad, "temperature": temperature,
            "rest": rest, "ragged": ragged, "train": train}


def _sample(rows, vocab, *, x="f32", pad=0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    return {"op": "sample", "rows": rows, "vocab": vocab, "x": x, "pad": pad, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed}


def listed():
    named = {
        # a training batch of the ten-class classifier taught by a larger one: the smallest step, latency
        "distill_classes": _distill(512, 10, 5, temperature=2.0),
        # logits as wide as the large layer, its batch
        "distill_wide_f32": _distill(8192, 4096, 32, temperature=2.0),
        # a training batch over a large vocabulary: the largest
        "distill_large_bf16": _distill(4096, 131072, 64, x="bf16"),
        # odd vocabulary (rows start off 16-byte boundaries), lists of different lengths, masked rows, no rest
        "distill_ragged_f32": _distill(1000, 50001, 33, rest=False, ragged=True),
        # validation: the loss alone, no gradient asked for
        "distill_eval_f16": _distill(2048, 32768, 16, x="f16", temperature=1.5, train=False),
        # a teacher's record of a training batch over a large vocabulary
        "top_large_bf16": _top(4096, 131072, 64, x="bf16"),
        # the record of a few prompts: latency
        "top_few_f32": _top(4, 32768, 8, temperature=2.0),
        # long lists of an odd vocabulary that is padded in memory
        "top_odd_f16": _top(777, 100003, 256, x="f16", pad=29),
        # serving one sequence: the next token
        "sample_one_bf16": _sample(1, 131072, x="bf16", temperature=0.8, top_k=50, top_p=0.9),
        # serving a full batch of requests, each with its own parameters
        "sample_mixed_bf16": _sample(256, 131072, x="bf16", mixed=True),
        # nucleus sampling alone: the whole row's mass decides
        "sample_nucleus_f32": _sample(64, 50001, top_p=0.95, temperature=0.9),
        # rollouts from the untruncated distribution
        "sample_plain_f16": _sample(1000, 32768, x="f16"),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("top", "distill", "sample"))
    vocab = _spread(rng, 10, 200000)
    most = {"top": 2**28, "distill": 2**28, "sample": 2**25}[op]
    rows = _spread(rng, 1, max(1, min(8192 if op != "sample" else 1024, most // vocab)))
    x = rng.choice(("f32", "bf16", "f16"))
    pad = rng.choice((0, 0, rng.randrange(1, 100)))
    temperature = rng.choice((1.0, round(rng.uniform(0.5, 4.0), 2)))
    k = _spread(rng, 1, min(vocab, 256))
    if op == "top":
        return _top(rows, vocab, k, x=x, pad=pad, temperature=temperature)
    if op == "distill":
        return _distill(rows, vocab, k, x=x, pad=pad, temperature=temperature, rest=rng.random() < 0.6,
                        ragged=rng.random() < 0.4, train=rng.random() < 0.75)
    if rng.random() < 0.3:
        return _sample(rows, vocab, x=x, pad=pad, mixed=True)
    return _sample(rows, vocab, x=x, pad=pad, temperature=temperature, top_k=rng.choice((0, k)),
                   top_p=rng.choice((1.0, round(rng.uniform(0.5, 0.99), 2))),
                   min_p=rng.choice((0.0, round(rng.uniform(0.01, 0.2), 3))))


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEVICE)


def _logits(gen, rows, vocab):
    x = torch.randn(rows, vocab, generator=gen, device=DEVICE).mul_(2.0)
    raised = min(32, vocab // 4)
    if raised:
        at = torch.randint(0, vocab, (rows, raised), generator=gen, device=DEVICE)
        x.scatter_add_(1, at, 4.0 + 12.0 * _rand(gen, rows, raised) * _rand(gen, rows, 1))
    return x


def _stored(x, case):
    """x in the case's type, as the first columns of rows of vocab + pad."""
    full = torch.zeros(case["rows"], case["vocab"] + case["pad"], device=DEVICE, dtype=DTYPES[case["x"]])
    full[:, :case["vocab"]] = x
    return full[:, :case["vocab"]]


def prepare(case, seed):
    gen = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    state = {"case": {k: v for k, v in case.items() if k != "name"}}
    x = _logits(gen, rows, vocab)
    if case["op"] == "top":
        state["logits"] = _stored(x, case)
    elif case["op"] == "distill":
        values, indices = torch.topk(x, case["k"], dim=1)
        values = values.to(DTYPES[case["x"]])
        state["log_rest"] = state["weights"] = None
        if case["rest"]:
            others = x.scatter(1, indices, -math.inf) / case["temperature"]
            state["log_rest"] = torch.logsumexp(others, 1)
            del others
        if case["ragged"]:
            kept = torch.randint(1, case["k"] + 1, (rows, 1), generator=gen, device=DEVICE)
            kept = torch.where(_rand(gen, rows, 1) < 0.7, torch.full_like(kept, case["k"]), kept)
            kept = torch.where(_rand(gen, rows, 1) < 0.02, torch.zeros_like(kept), kept)
            indices = torch.where(torch.arange(case["k"], device=DEVICE) < kept, indices, -1)
            # a row always counts for something: the first one's weight is one
            state["weights"] = torch.where(_rand(gen, rows) < 0.3, torch.zeros(rows, device=DEVICE), 0.5 + _rand(gen, rows))
            state["weights"][0] = 1.0
        state["values"], state["indices"] = values, indices
        student = x.mul_(0.8).add_(torch.randn(rows, vocab, generator=gen, device=DEVICE))
        state["logits"] = _stored(student, case).requires_grad_(case["train"])
    else:
        state["logits"] = _stored(x, case)
        state["uniforms"] = _rand(gen, rows)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            state[name] = case[name]
        if case["mixed"]:
            off = _rand(gen, 3, rows) < torch.tensor([[0.3], [0.3], [0.6]], device=DEVICE)
            state["temperature"] = torch.where(_rand(gen, rows) < 0.1, torch.zeros(rows, device=DEVICE), 0.5 + _rand(gen, rows))
            state["top_k"] = torch.where(off[0], 0, torch.randint(1, 101, (rows,), generator=gen, device=DEVICE)).to(torch.int32)
            state["top_p"] = torch.where(off[1], torch.ones(rows, device=DEVICE), 0.5 + 0.49 * _rand(gen, rows))
            state["min_p"] = torch.where(off[2], torch.zeros(rows, device=DEVICE), 0.2 * _rand(gen, rows))
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return {"top": _own_top, "distill": _own_distill, "sample": _own_sample}[op](state)
    return {"top": _plain_top, "distill": _plain_distill, "sample": _plain_sample}[op](state)


def _own_top(state):
    from tropnn_amd import top_logits

    got = top_logits(state["logits"], state["case"]["k"], temperature=state["case"]["temperature"])
    return {"values": got.values, "indices": got.indices, "log_rest": got.log_rest}


def _own_distill(state):
    from tropnn_amd import distillation_loss

    logits = state["logits"]
    logits.grad = None
    loss = distillation_loss(logits, state["values"], state["indices"], state["log_rest"], weights=state["weights"],
                             temperature=state["case"]["temperature"])
    if not state["case"]["train"]:
        return {"loss": loss}
    loss.backward()
    return {"loss": loss.detach(), "grad": logits.grad}


def _own_sample(state):
    from tropnn_amd import sample_tokens

    got = sample_tokens(state["logits"], state["uniforms"], temperature=state["temperature"], top_k=state["top_k"],
                        top_p=state["top_p"], min_p=state["min_p"])
    return {"tokens": got.tokens, "log_probs": got.log_probs}


def _log_sum_exp(z):
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    return m + torch.log(torch.exp(z - m).sum(1, keepdim=True))


def _plain_top(state):
    case, logits = state["case"], state["logits"]
    x = logits.float()
    order, at = torch.sort(x, dim=1, descending=True, stable=True)
    at = at[:, :case["k"]]
    rest = _log_sum_exp(order[:, case["k"]:] * (1.0 / case["temperature"])) if case["k"] < case["vocab"] else None
    return {"values": logits.gather(1, at), "indices": at.contiguous(),
            "log_rest": rest[:, 0] if rest is not None else torch.full_like(x[:, 0], -math.inf)}


def _plain_distill(state):
    case, t = state["case"], state["case"]["temperature"]
    logits = state["logits"].detach()
    rows, vocab = logits.shape
    listed_ = state["indices"] >= 0
    at = torch.where(listed_, state["indices"], vocab)  # what is not listed goes to a column past the end
    z = torch.cat((logits.float() * (1.0 / t), torch.full((rows, 1), -math.inf, device=DEVICE)), 1)
    v = torch.where(listed_, state["values"].float() * (1.0 / t), -math.inf)
    some = listed_.any(1, keepdim=True)
    lse = _log_sum_exp(z)
    log_z = _log_sum_exp(v if state["log_rest"] is None else torch.cat((v, state["log_rest"][:, None]), 1))
    log_p = torch.where(listed_, v - log_z, 0.0)
    p = torch.where(listed_, torch.exp(v - log_z), 0.0)
    log_q = torch.where(listed_, z.gather(1, at) - lse, 0.0)
    loss = (p * (log_p - log_q)).sum(1, keepdim=True)
    share = torch.ones_like(loss)  # of its q, what a logit outside the list has as its gradient
    if state["log_rest"] is not None:
        log_p0 = state["log_rest"][:, None] - log_z
        log_q0 = _log_sum_exp(z.scatter(1, at, -math.inf)) - lse
        loss = loss + torch.where(log_p0 > -math.inf, torch.exp(log_p0) * (log_p0 - log_q0), 0.0)
        share = torch.where(log_p0 > -math.inf, 1.0 - torch.exp(log_p0 - log_q0), 1.0)
    weight = torch.ones(rows, 1, device=DEVICE) if state["weights"] is None else state["weights"][:, None]
    used = some & (weight != 0)
    loss = (torch.where(used, t * t * loss, 0.0) * weight).sum() / weight.sum()
    if not case["train"]:
        return {"loss": loss}
    grad = torch.exp(z - lse) * share
    grad.scatter_(1, at, torch.exp(log_q) - p)
    grad = torch.where(used, grad * (t * weight / weight.sum()), 0.0)
    return {"loss": loss, "grad": grad[:, :vocab].to(logits.dtype)}


def _column(value, like, dtype):
    return value[:, None].to(dtype) if isinstance(value, torch.Tensor) else torch.full_like(like, value, dtype=dtype)


def _plain_sample(state):
    x = state["logits"].float()
    rows, vocab = x.shape
    u = state["uniforms"][:, None]
    temperature, top_p, min_p = (_column(state[n], u, torch.float32) for n in ("temperature", "top_p", "min_p"))
    top_k = _column(state["top_k"], u, torch.int64)
    greedy = temperature <= 0
    m = x.amax(1, keepdim=True)
    # weights in units of 2^-40 of the largest: whole numbers, whose sums are exact in any order
    inverse = torch.full_like(temperature, 1.4426950408889634) / torch.where(greedy, 1.0, temperature)
    weight = torch.exp2((x - m) * inverse)
    w = (weight * FIXED).to(torch.int64)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    w_sorted, weight_sorted = w.gather(1, order), weight.gather(1, order)
    rank = torch.arange(vocab, device=DEVICE)[None]
    w_sorted = torch.where((rank < top_k) | (top_k <= 0), w_sorted, 0)
    running = w_sorted.cumsum(1)
    total = running[:, -1:]
    limit = torch.where(top_p < 1.0, (top_p.double() * total.double()).to(torch.int64).clamp(min=1), total)
    kept = (running - w_sorted < limit) & (weight_sorted >= min_p.clamp(max=1.0))
    w_kept = torch.zeros_like(w).scatter(1, order, torch.where(kept, w_sorted, 0))
    running = w_kept.cumsum(1)
    total = running[:, -1:]
    target = torch.minimum((u.double() * total.double()).to(torch.int64), total - 1)
    token = (running <= target).sum(1, keepdim=True)
    token = torch.where(greedy, order[:, :1], token)
    log_prob = torch.log(w_kept.gather(1, token).float() / total.float())
    return {"tokens": token[:, 0], "log_probs": torch.where(greedy, 0.0, log_prob)[:, 0]}


def work(case):
    e, n = SIZES[case["x"]], case["rows"] * case["vocab"]
    read, written = n * e, 0
    if case["op"] == "top":
        written = case["rows"] * (case["k"] * (e + 8) + 4)
    elif case["op"] == "distill":
        read += case["rows"] * (case["k"] * (e + 8) + 4 * case["rest"] + 4 * case["ragged"])
        written = 4 + (n * e if case["train"] else 0)
    else:
        read += case["rows"] * (20 if case["mixed"] else 4)
        written = case["rows"] * 12
    # an exponential, a product and two sums a logit; the gradient takes as many again
    return {"bytes": read + written, "flops": n * (8 if case["op"] == "distill" and case["train"] else 4)}


def exact(case, seed):
    state = prepare(case, seed)
    return {"top": _exact_top, "distill": _exact_distill, "sample": _exact_sample}[case["op"]](state)


def _exact_top(state):
    k, t = state["case"]["k"], state["case"]["temperature"]
    rest = []
    for x in state["logits"].split(512):
        low = torch.sort(x.double(), dim=1, descending=True, stable=True).values[:, k:] / t
        rest.append(torch.logsumexp(low, 1) if low.shape[1] else torch.full((len(x),), -math.inf, device=DEVICE, dtype=torch.float64))
    return {"values": None, "indices": None, "log_rest": torch.cat(rest)}


def _exact_distill(state):
    """Sum of p log(p / q) over the listed logits and the rest as one class more; its gradient, class by class."""
    case, t = state["case"], state["case"]["temperature"]
    rows = case["rows"]
    weight = torch.ones(rows, device=DEVICE, dtype=torch.float64) if state["weights"] is None else state["weights"].double()
    total, losses, grads = weight.sum(), [], []
    for lo in range(0, rows, 512):
        part = slice(lo, min(rows, lo + 512))
        z = state["logits"].detach()[part].double() / t
        at = state["indices"][part]
        there = at >= 0
        safe = at.clamp(min=0)
        teacher = (state["values"][part].double() / t).masked_fill(~there, -math.inf)
        if state["log_rest"] is not None:
            teacher = torch.cat((teacher, state["log_rest"][part, None].double()), 1)
        p = torch.softmax(teacher, 1)
        log_q_all = torch.log_softmax(z, 1)
        mask = torch.zeros_like(z, dtype=torch.bool)
        mask.scatter_(1, torch.where(there, safe, at[:, :1].clamp(min=0)), there.any(1, keepdim=True).expand_as(at))
        log_q = log_q_all.gather(1, safe)
        if state["log_rest"] is not None:
            log_q = torch.cat((log_q, torch.logsumexp(log_q_all.masked_fill(mask, -math.inf), 1, keepdim=True)), 1)
        here = (p > 0) & torch.isfinite(p)
        kl = torch.where(here, p * (torch.log(torch.where(here, p, 1.0)) - torch.where(here, log_q, 0.0)), 0.0).sum(1)
        w = weight[part] * there.any(1)
        losses.append((w * t * t * kl).sum())
        if case["train"]:
            q = torch.exp(log_q_all)
            g = q.clone()
            if state["log_rest"] is not None:
                p0, q0 = p[:, -1:], torch.exp(log_q[:, -1:])
                g = torch.where(mask, q, q * torch.where(p0 > 0, 1.0 - p0 / q0, 1.0))
            g.scatter_add_(1, safe, -torch.where(there, p[:, :at.shape[1]], 0.0))
            grads.append(torch.where(w[:, None] > 0, g * (t * w / total)[:, None], 0.0))
    out = {"loss": torch.stack(losses).sum() / total}
    return dict(out, grad=torch.cat(grads)) if case["train"] else out


def _exact_sample(state):
    x = state["logits"].double()
    u = state["uniforms"].double()[:, None]
    temperature, top_p, min_p = (_column(state[n], u, torch.float64) for n in ("temperature", "top_p", "min_p"))
    top_k = _column(state["top_k"], u, torch.int64)
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ordered - ordered[:, :1]) / temperature)
    rank = torch.arange(x.shape[1], device=DEVICE)[None]
    w = torch.where((rank < top_k) | (top_k <= 0), w, 0.0)
    before = w.cumsum(1) - w
    kept = (rank == 0) | (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1.0)
    w = torch.where(kept & (w >= min_p), w, 0.0)
    by_index = torch.zeros_like(w).scatter(1, order, w)
    running = by_index.cumsum(1)
    token = (running <= u * running[:, -1:]).sum(1, keepdim=True).clamp(max=x.shape[1] - 1)
    log_prob = torch.log(by_index.gather(1, token) / running[:, -1:])
    return {"tokens": None, "log_probs": torch.where(temperature > 0, log_prob, 0.0)[:, 0]}
