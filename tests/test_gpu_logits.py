"""top_logits, distillation_loss and sample_tokens on the GPU against plain
forms in 64 bits on the CPU.

Tolerances, from f32 arithmetic (u = 2^-24): an exponential 2^a with |a| <= 40
carries the rounding of a (two operations, 80 u) and of the instruction (u); a
sum of n positive terms in a tree of per-thread runs adds at most (n / 64 + 16)
u, 2e-5 for the sizes here. So a probability is within 3e-5 of its value, a
log-sum within 3e-5 absolute (plus u per unit of its size), and what is stored
in 16 bits carries half an ulp more."""
from __future__ import annotations

import math

import pytest
import torch

from tropnn_amd import distillation_loss, sample_tokens, top_logits, unit_gradient
from tropnn_amd.backends.logits_hip import scale_in_place

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_ULP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
SMALLEST = {F32: 1e-38, F16: 2.0**-24, BF16: 1e-38}
REL = 3e-5
LOWEST = torch.finfo(F32).min


def rows_of(rows, vocab, dtype, seed, *, pad=0, shift=0, scale=3.0):
    """Logits [rows, vocab] on the GPU as a slice: `pad` columns between rows,
    `shift` elements before the first."""
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=gen) * scale).to(dtype)
    flat = torch.zeros(shift + rows * (vocab + pad), dtype=dtype, device=DEV)
    view = flat[shift:].view(rows, vocab + pad)[:, :vocab]
    view.copy_(x)
    return view


def order_of(x):
    """The order of a row's logits (CPU), and the logits in it."""
    return torch.sort(x.double() + 0.0, dim=-1, descending=True, stable=True)


def check_top(logits, k, temperature=1.0):
    got = top_logits(logits, k, temperature=temperature)
    x = logits.detach().cpu()
    values, indices = order_of(x)
    assert got.indices.dtype == torch.int64 and got.values.dtype == logits.dtype and got.log_rest.dtype == F32
    assert torch.equal(got.indices.cpu(), indices[..., :k])
    assert torch.equal(got.values.cpu().nan_to_num(7e4), x.gather(-1, indices[..., :k]).nan_to_num(7e4))
    rest = values[..., k:] / temperature
    want = torch.logsumexp(rest, -1) if rest.shape[-1] else torch.full(x.shape[:-1], -math.inf, dtype=torch.float64)
    have = got.log_rest.cpu().double()
    plain = torch.isfinite(want) & (want.abs() < 1e38)
    assert torch.equal(torch.isnan(have), torch.isnan(want))
    assert torch.equal(have[~plain & (want.abs() == math.inf)], want[~plain & (want.abs() == math.inf)])
    assert ((have - want).abs()[plain] <= REL * (1 + want.abs()[plain])).all(), (have, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize(
    "rows,vocab,k,pad,shift",
    [
        (1, 1, 1, 0, 0),
        (3, 2, 2, 0, 1),
        (5, 10, 3, 0, 0),
        (4, 63, 63, 2, 0),
        (2, 1000, 1, 5, 3),
        (2, 1000, 1000, 0, 0),
        (3, 4099, 1024, 1, 7),
        (300, 777, 17, 0, 0),
        (2, 20001, 256, 3, 1),
        (3, 70001, 50, 0, 0),
        (1, 131072, 64, 0, 0),
        (2, 200003, 200, 0, 5),
    ],
)
def test_top_logits(rows, vocab, k, pad, shift, dtype):
    check_top(rows_of(rows, vocab, dtype, rows + vocab, pad=pad, shift=shift), k, temperature=1.0 if vocab % 2 else 1.7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [9, 1000, 33000])
def test_top_logits_ties_and_special_values(vocab, dtype):
    """Few different values, equal rows, masks, infinities, NaN and both zeros."""
    gen = torch.Generator().manual_seed(vocab)
    few = torch.randint(-3, 3, (vocab,), generator=gen).float()
    low = torch.finfo(dtype).min
    rows = [few, torch.zeros(vocab), torch.full((vocab,), -math.inf), torch.full((vocab,), low)]
    rows.append(torch.where(torch.rand(vocab, generator=gen) < 0.5, 0.0, -0.0))
    masked = torch.full((vocab,), -math.inf)
    masked[vocab // 2] = 1.0
    rows.append(masked)
    rows.append(torch.where(torch.rand(vocab, generator=gen) < 0.9, low, 2.0))
    nan = few.clone()
    nan[vocab // 3] = math.nan
    rows.append(nan)
    top = few.clone()
    top[vocab // 4] = math.inf
    rows.append(top)
    rows.append(torch.arange(vocab).float())  # rising: every later logit is better than all before
    rows.append(-torch.arange(vocab).float())
    x = torch.stack(rows).to(dtype).to(DEV)
    for k in (1, 4, min(vocab, 900)):
        check_top(x, k)


def test_top_logits_leading_dimensions_and_layouts():
    base = rows_of(6, 500, F32, 1).reshape(2, 3, 500)
    check_top(base, 7)
    check_top(base[:, 1], 7)  # rows 1500 apart
    check_top(base[:, ::2, 3:450], 7)
    check_top(base.transpose(1, 2).contiguous().transpose(1, 2), 7)  # classes not contiguous: copied
    check_top(base[0, 0], 7)
    check_top(base[:, :1].expand(2, 3, 500), 7)
    empty = top_logits(torch.empty(0, 12, device=DEV), 3)
    assert empty.values.shape == (0, 3) and empty.indices.shape == (0, 3) and empty.log_rest.shape == (0,)


def distill_reference(logits, values, indices, log_rest, weights, t, scale=1.0, mean=True):
    """Loss and gradient in 64 bits, and the gradient's tolerance."""
    x = logits.detach().cpu().double()
    vocab = x.shape[-1]
    x = x.reshape(-1, vocab)
    rows, k = x.shape[0], values.shape[-1]
    v, at = values.cpu().double().reshape(rows, k), indices.cpu().reshape(rows, k)
    rest = None if log_rest is None else log_rest.cpu().double().reshape(rows)
    w = torch.ones(rows, dtype=torch.float64) if weights is None else weights.cpu().double().reshape(rows)
    d = w.sum() if mean else torch.tensor(1.0, dtype=torch.float64)
    loss, grad, bound = torch.tensor(0.0, dtype=torch.float64), torch.zeros_like(x), torch.zeros_like(x)
    for r in range(rows):
        here = at[r] >= 0
        if w[r] == 0 or not here.any():
            continue
        idx, teacher = at[r][here], v[r][here] / t
        if rest is not None:
            teacher = torch.cat((teacher, rest[r].reshape(1)))
        log_p = torch.log_softmax(teacher, 0)
        log_q_all = torch.log_softmax(x[r] / t, 0)
        listed = torch.zeros(vocab, dtype=torch.bool)
        listed[idx] = True
        log_q = log_q_all[idx]
        if rest is not None:
            others = log_q_all[~listed]
            log_q0 = torch.logsumexp(others, 0) if len(others) else torch.tensor(-math.inf, dtype=torch.float64)
            log_q = torch.cat((log_q, log_q0.reshape(1)))
        p = log_p.exp()
        terms = torch.where(p > 0, p * (log_p - log_q), 0.0)
        loss = loss + w[r] * t * t * terms.sum()
        q = log_q_all.exp()
        g, b = q.clone(), q.clone()
        if rest is not None:
            ratio = torch.where(p[-1] > 0, p[-1] / log_q[-1].exp(), 0.0)
            g[~listed] *= 1 - ratio
            b[~listed] *= 1 + ratio
        g[idx] -= p[: len(idx)]
        b[idx] += p[: len(idx)]
        coef = t * scale * w[r] / d
        grad[r] = coef * g
        bound[r] = coef.abs() * REL * b + HALF_ULP[logits.dtype] * grad[r].abs() + SMALLEST[logits.dtype]
    return scale * loss / d, grad.reshape(logits.shape), bound.reshape(logits.shape)


def make_record(rows, vocab, k, seed, *, values_dtype=F32, t=1.0, rest=True):
    gen = torch.Generator().manual_seed(seed)
    teacher = torch.randn(rows, vocab, generator=gen) * 3
    values, indices = order_of(teacher)
    log_rest = None
    if rest:
        log_rest = (torch.logsumexp(values[:, k:] / t, 1) if k < vocab else torch.full((rows,), -math.inf)).float().to(DEV)
    return values[:, :k].to(values_dtype).to(DEV), indices[:, :k].contiguous().to(DEV), log_rest


def check_distill(logits, values, indices, log_rest, weights=None, t=1.0, **kw):
    want, want_grad, bound = distill_reference(logits, values, indices, log_rest, weights, t,
                                               kw.get("scale", 1.0), kw.get("reduction", "mean") == "mean")
    x = logits.detach().requires_grad_(True)
    loss = distillation_loss(x, values, indices, log_rest, weights=weights, temperature=t, **kw)
    assert loss.shape == () and loss.dtype == F32
    loss.backward()
    got = float(loss.detach())
    if math.isinf(want) or math.isnan(want):
        assert str(got) == str(float(want))
    else:
        assert abs(got - float(want)) <= REL * abs(float(want)) + REL * abs(kw.get("scale", 1.0)) * t * t * max(1, logits.numel() // logits.shape[-1] if kw.get("reduction") == "sum" else 1), (got, float(want))
    assert x.grad.dtype == logits.dtype and x.grad.shape == logits.shape
    off = (x.grad.cpu().double() - want_grad).abs() - bound
    assert (off <= 0).all(), (off.max(), x.grad, want_grad)
    with torch.no_grad():  # without a gradient: the same loss
        again = distillation_loss(logits, values, indices, log_rest, weights=weights, temperature=t, **kw)
    assert abs(float(again) - got) <= 1e-5 * abs(got) or str(float(again)) == str(got)
    return loss.detach(), x.grad


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize(
    "rows,vocab,k,pad,shift,t",
    [
        (1, 1, 1, 0, 0, 1.0),
        (3, 2, 1, 0, 1, 2.0),
        (512, 10, 4, 0, 0, 2.0),
        (7, 63, 63, 3, 0, 0.7),
        (9, 130, 9, 0, 0, 1.0),
        (5, 2049, 300, 1, 3, 3.0),
        (2, 4096, 1024, 0, 0, 1.0),
        (33, 5003, 33, 0, 1, 1.0),
        (3, 33001, 64, 7, 0, 1.3),
        (2, 131072, 16, 0, 0, 1.0),
        (1, 200003, 5, 0, 0, 1.0),
    ],
)
def test_distillation(rows, vocab, k, pad, shift, t, rest, dtype):
    logits = rows_of(rows, vocab, dtype, vocab, pad=pad, shift=shift)
    values, indices, log_rest = make_record(rows, vocab, k, rows, t=t, rest=rest, values_dtype=dtype)
    check_distill(logits, values, indices, log_rest, t=t)


@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("vocab", [12, 700, 9000])
def test_distillation_ragged_lists_and_weights(vocab, rest):
    rows, k = 11, 9
    logits = rows_of(rows, vocab, F32, 5)
    values, indices, log_rest = make_record(rows, vocab, k, 6, rest=rest)
    indices[1, 4:] = -1
    indices[2, :] = -1  # no list: no loss, no gradient
    indices[3, ::2] = -5
    weights = torch.linspace(0.1, 2.0, rows, device=DEV)
    weights[5] = 0.0
    logits[5] = math.nan  # left out, whatever it holds
    values[5] = math.inf
    for kw in ({}, {"reduction": "sum"}, {"scale": 0.25}):
        _, grad = check_distill(logits, values, indices, log_rest, weights, **kw)
        assert not grad[5].any() and not grad[2].any()
    check_distill(logits[:5], values[:5], indices[:5], None if log_rest is None else log_rest[:5])


@pytest.mark.parametrize("dtype", [F32, F16])
def test_distillation_masked_logits(dtype):
    """-inf and the lowest value among the student's and the teacher's logits."""
    vocab, k = 600, 8
    low = torch.finfo(dtype).min
    logits = rows_of(6, vocab, dtype, 3)
    values, indices, log_rest = make_record(6, vocab, k, 4, values_dtype=dtype)
    outside = torch.ones(vocab, dtype=torch.bool, device=DEV)
    outside[indices[0]] = False
    logits[0, torch.nonzero(outside)[:200, 0]] = -math.inf
    logits[1, :] = low  # all masked with the lowest value: uniform
    logits[2, 100:] = low
    values[3, 5:] = -math.inf  # a teacher with fewer than k classes left
    log_rest[3] = -math.inf
    values[4, 5:] = low
    log_rest[4] = LOWEST
    if dtype == F16:
        logits[2, 100:] = 0  # the lowest f16 leaves probabilities that f32 holds, with infinite-looking losses
    for lr in (log_rest, None):
        check_distill(logits[[0, 1, 3, 4, 5]], values[[0, 1, 3, 4, 5]], indices[[0, 1, 3, 4, 5]],
                      None if lr is None else lr[[0, 1, 3, 4, 5]])
    # mass where the student has none: an infinite loss, a gradient that is still the formula's
    gone = logits[5:6].clone()
    gone[0, indices[5, 0]] = -math.inf
    loss, grad = check_distill(gone, values[5:6], indices[5:6], None)
    assert float(loss) == math.inf and torch.isfinite(grad).all()


def test_distillation_bad_rows_are_nan_and_stay_apart():
    logits = rows_of(4, 300, F32, 8)
    values, indices, log_rest = make_record(4, 300, 5, 9)
    logits[0, 7] = math.nan
    indices[1, 2] = 300  # no such class
    logits[2, :] = -math.inf
    x = logits.requires_grad_(True)
    loss = distillation_loss(x, values, indices, log_rest)
    loss.backward()
    assert math.isnan(float(loss.detach()))
    _, want, bound = distill_reference(logits[3:].detach(), values[3:], indices[3:], log_rest[3:], None, 1.0)
    off = (x.grad[3:].cpu().double() - want / 4).abs() - bound / 4
    assert (off <= 0).all() and not torch.isfinite(x.grad[:3]).all(1).any()


def test_distillation_no_rows_and_no_weight():
    values, indices, log_rest = make_record(3, 40, 5, 2)
    x = rows_of(3, 40, F32, 1).requires_grad_(True)
    zero = torch.zeros(3, device=DEV)
    loss = distillation_loss(x, values, indices, log_rest, weights=zero)
    loss.backward()
    assert math.isnan(float(loss.detach())) and not x.grad.any()
    assert float(distillation_loss(x, values, indices, log_rest, weights=zero, reduction="sum").detach()) == 0.0
    e = torch.empty(0, 40, device=DEV, requires_grad=True)
    loss = distillation_loss(e, values[:0], indices[:0], log_rest[:0])
    loss.backward()
    assert math.isnan(float(loss.detach())) and e.grad.shape == (0, 40)
    assert float(distillation_loss(e, values[:0], indices[:0], reduction="sum").detach()) == 0.0


@pytest.mark.parametrize("rest", [True, False])
def test_distillation_gradient_against_differences(rest):
    """Differences of the 64-bit loss along a direction, and of the kernel's
    own loss along one (f32: a step of 0.05 carries 0.05^2 of curvature and
    2 * 3e-5 / 0.05 of rounding)."""
    logits = rows_of(3, 400, F32, 1)
    values, indices, log_rest = make_record(3, 400, 7, 2, t=2.0, rest=rest)
    _, grad = check_distill(logits, values, indices, log_rest, t=2.0)
    d = torch.randn(3, 400, generator=torch.Generator().manual_seed(3))
    slope = float((grad.cpu().double() * d).sum())
    h = 1e-4


    def loss64(step):
        return float(distill_reference((logits.cpu().double() + step * d), values, indices, log_rest, None, 2.0)[0])

    HALF_ULP[torch.float64], SMALLEST[torch.float64] = 0.0, 0.0
    assert abs((loss64(h) - loss64(-h)) / (2 * h) - slope) <= 1e-4 * max(1.0, abs(slope))

    def loss32(step):
        return float(distillation_loss(logits + step * d.to(DEV), values, indices, log_rest, temperature=2.0))

    assert abs((loss32(0.05) - loss32(-0.05)) / 0.1 - slope) <= 5e-3 * max(1.0, abs(slope))


def test_distillation_incoming_gradients():
    """One, the kept unit, another value, a sum of losses, a second backward
    through the same graph; logits that are shared by broadcasting."""
    values, indices, log_rest = make_record(4, 257, 6, 2)
    logits = rows_of(4, 257, F32, 1)

    def grad_of(run):
        x = logits.clone().requires_grad_(True)
        run(x, distillation_loss(x, values, indices, log_rest))
        return x.grad

    want = grad_of(lambda x, loss: loss.backward())
    assert torch.equal(grad_of(lambda x, loss: loss.backward(unit_gradient(loss))), want)
    assert torch.allclose(grad_of(lambda x, loss: (2.5 * loss).backward()), 2.5 * want, rtol=1e-6, atol=0)
    assert torch.allclose(grad_of(lambda x, loss: (loss + 0.5 * x.sum()).backward()), want + 0.5, rtol=1e-6)
    assert not grad_of(lambda x, loss: (0.0 * loss).backward()).any()

    def twice(x, loss):
        loss.backward(torch.tensor(3.0, device=DEV), retain_graph=True)
        loss.backward()

    assert torch.allclose(grad_of(twice), 4.0 * want, rtol=1e-5, atol=1e-9)
    one = logits[:1].clone().requires_grad_(True)
    distillation_loss(one.expand(4, 257), values, indices, log_rest).backward()
    rows = logits[:1].repeat(4, 1).requires_grad_(True)
    distillation_loss(rows, values, indices, log_rest).backward()
    assert torch.allclose(one.grad, rows.grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 7, 8, 4099])
def test_scale_in_place(n, dtype):
    x = torch.randn(n + 3, device=DEV).to(dtype)
    part = x[3:]
    want = (part.float() * 1.7).to(dtype)
    before = x[:3].clone()
    scale_in_place(part, torch.tensor(1.7, device=DEV))
    assert torch.equal(part, want) and torch.equal(x[:3], before)
    scale_in_place(part, torch.tensor(1.0, device=DEV))
    assert torch.equal(part, want)


# temperature log2(e) in f32 makes the exponents' factor exactly one, and whole
# logits then have weights that are exact powers of two: everything is decided
LOG2E = float(torch.tensor(1.4426950408889634, dtype=F32))
ONE = 1 << 40


def sample_reference(x, u, top_k=0, top_p=1.0, min_p=0.0):
    """Token and probability of a row of whole logits (Python numbers; None:
    -inf) at temperature log2(e), in whole numbers."""
    m = max(v for v in x if v is not None)
    w = [0 if v is None else (ONE >> min(m - v, 64)) for v in x]
    order = sorted((i for i in range(len(x))), key=lambda i: (-(x[i] if x[i] is not None else -1e9), i))
    kept = order[:top_k] if top_k > 0 else order
    if top_p < 1.0:
        limit = max(1, int(float(torch.tensor(top_p, dtype=F32)) * float(sum(w[i] for i in kept))))
        total, left = 0, []
        for i in kept:
            if total < limit:
                left.append(i)
            total += w[i]
        kept = left
    floor = min(float(torch.tensor(min_p, dtype=F32)), 1.0)
    kept = sorted(i for i in kept if w[i] >= floor * ONE)
    total = sum(w[i] for i in kept)
    target = min(int(float(torch.tensor(u, dtype=F32)) * float(total)), total - 1)
    running = 0
    for i in kept:
        running += w[i]
        if running > target:
            return i, w[i] / total
    raise AssertionError


PARAMETERS = [
    dict(),
    dict(top_k=1),
    dict(top_k=5),
    dict(top_k=100),
    dict(top_k=10**6),
    dict(top_p=0.5),
    dict(top_p=0.9),
    dict(top_p=0.999),
    dict(top_p=1e-6),
    dict(min_p=0.125),
    dict(min_p=0.1),
    dict(min_p=1.0),
    dict(top_k=40, top_p=0.8),
    dict(top_k=7, min_p=0.3),
    dict(top_p=0.7, min_p=0.01),
    dict(top_k=30, top_p=0.95, min_p=0.05),
    dict(top_k=900, top_p=0.99),
    dict(top_k=2000, top_p=0.9),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab,low", [(1, -5), (10, -4), (200, -8), (5000, -20), (5000, -1), (40003, -9), (40003, -60)])
def test_sample_exact(vocab, low, dtype):
    """Whole logits: many ties, and sums whose every value is known."""
    gen = torch.Generator().manual_seed(vocab)
    rows = 4
    x = torch.randint(low, 1, (rows, vocab), generator=gen)
    x[1] = -(x[1].abs() ** 0.5).long() * 4  # fewer different values
    hidden = torch.rand(rows, vocab, generator=gen) < 0.3
    hidden[:, 0] = False
    logits = torch.where(hidden, -math.inf, x.float()).to(dtype).to(DEV)
    lists = [[None if h else int(v) for v, h in zip(a, b)] for a, b in zip(x.tolist(), hidden.tolist())]
    for n, kw in enumerate(PARAMETERS):
        u = torch.rand(rows, generator=gen)
        u[0] = (0.0, 1.0 - 2.0**-24, 0.5)[n % 3]
        got = sample_tokens(logits, u.to(DEV), temperature=LOG2E, **kw)
        want = [sample_reference(r, float(v), **kw) for r, v in zip(lists, u)]
        assert got.tokens.tolist() == [w[0] for w in want], kw
        probs = torch.tensor([w[1] for w in want], dtype=torch.float64)
        assert torch.allclose(got.log_probs.cpu().double(), probs.log(), rtol=1e-6, atol=1e-6), kw


def test_sample_per_row_parameters_match_scalars():
    """A row's answer does not depend on the batch around it."""
    rows = len(PARAMETERS)
    logits = rows_of(rows, 3001, BF16, 4)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(1)).to(DEV)
    temperature = torch.linspace(0.4, 2.0, rows)
    temperature[3] = 0.0
    values = {n: torch.tensor([float(kw.get(n, d)) for kw in PARAMETERS]) for n, d in (("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    for kind in (torch.int32, torch.int64):
        together = sample_tokens(logits, u, temperature=temperature.to(DEV), top_k=values["top_k"].to(kind).to(DEV),
                                 top_p=values["top_p"].to(DEV), min_p=values["min_p"].to(DEV))
        for r, kw in enumerate(PARAMETERS):
            alone = sample_tokens(logits[r], u[r], temperature=float(temperature[r]), **kw)
            assert alone.tokens.shape == ()
            assert int(alone.tokens) == int(together.tokens[r]) and float(alone.log_probs) == float(together.log_probs[r]), (r, kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [77, 50001])
@pytest.mark.parametrize("kw", PARAMETERS[:2] + PARAMETERS[5:7] + PARAMETERS[9:11] + PARAMETERS[12:16])
def test_sample_against_64_bits(vocab, dtype, kw):
    """The token's share of the distribution function holds its number, within
    what f32 weights move it by; its log-probability is the distribution's."""
    rows, t = 40, 0.8
    logits = rows_of(rows, vocab, dtype, 11, shift=1)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(5))
    got = sample_tokens(logits, u.to(DEV), temperature=t, **kw)
    x = logits.cpu().double()
    values, order = order_of(x)
    w = torch.exp((values - values[:, :1]) / t)
    rank = torch.arange(vocab)
    if kw.get("top_k", 0) > 0:
        w = torch.where(rank < kw["top_k"], w, 0.0)
    before = w.cumsum(1) - w
    limit = kw.get("top_p", 1.0) * w.sum(1, keepdim=True)
    kept = (rank == 0) | (before < limit) if kw.get("top_p", 1.0) < 1 else torch.ones_like(w, dtype=torch.bool)
    # a cut that f32 may place elsewhere: nothing to compare there
    near = ((before - limit).abs() < 1e-4 * limit).any(1) if kw.get("top_p", 1.0) < 1 else torch.zeros(rows, dtype=torch.bool)
    near |= ((w - kw.get("min_p", 0.0)).abs() < 1e-5).any(1) & (kw.get("min_p", 0.0) > 0)
    w = torch.where(kept & (w >= kw.get("min_p", 0.0)), w, 0.0)
    by_index = torch.zeros_like(w).scatter(1, order, w)
    by_index /= by_index.sum(1, keepdim=True)
    upto = by_index.cumsum(1)
    token = got.tokens.cpu()[:, None]
    p = by_index.gather(1, token)[:, 0]
    high, ok = upto.gather(1, token)[:, 0], ~near
    assert ok.any()
    assert (p[ok] > 0).all()
    assert ((u.double() <= high + 3e-5) & (u.double() >= high - p - 3e-5))[ok].all()
    assert torch.allclose(got.log_probs.cpu().double()[ok], p[ok].log(), rtol=REL, atol=REL)


def test_sample_special_rows():
    vocab = 500
    x = rows_of(8, vocab, F32, 3)
    x[0] = -math.inf
    x[1, 7] = math.nan
    x[2] = LOWEST  # all masked with the lowest value: uniform
    x[3, 9] = math.inf
    x[3, 99] = math.inf
    x[4] = -math.inf
    x[4, 321] = -2.0
    x[5, 250:] = LOWEST
    x[6] = -0.0
    x[6, 100:] = 0.0
    u = torch.full((8,), 0.75, device=DEV)
    for kw in ({}, {"top_k": 400}, {"top_p": 0.95}, {"top_k": 400, "top_p": 0.95}, {"min_p": 0.5}):
        got = sample_tokens(x, u, **kw)
        tokens, lp = got.tokens.tolist(), got.log_probs.tolist()
        assert tokens[0] == -1 and math.isnan(lp[0]) and tokens[1] == -1 and math.isnan(lp[1])
        n = min(kw.get("top_k", vocab), vocab)
        if kw.get("top_p", 1.0) < 1:
            n = math.ceil(n * 0.95)
        assert tokens[2] == int(0.75 * n) and abs(lp[2] + math.log(n)) < 1e-5
        assert tokens[3] == 99 and abs(lp[3] - math.log(0.5)) < 1e-6
        assert tokens[4] == 321 and lp[4] == 0.0
        assert 0 <= tokens[5] < 250
        assert tokens[6] == int(0.75 * n)
    cold = sample_tokens(x, u, temperature=0.0)
    want = [-1, -1, 0, 9, 321, int(x[5].argmax()), 0, int(x[7].argmax())]
    assert cold.tokens.tolist() == want and cold.log_probs.tolist()[2:] == [0.0] * 6
    tiny = sample_tokens(x, u, temperature=1e-30)
    assert tiny.tokens.tolist()[2] == 375 and tiny.tokens.tolist()[7] == want[7]
    none = sample_tokens(torch.empty(0, 9, device=DEV), torch.empty(0, device=DEV))
    assert none.tokens.shape == (0,) and none.log_probs.shape == (0,)


@pytest.mark.parametrize("op", ["top", "distill", "sample"])
def test_other_stream_and_graph_replays(op):
    """The same results on another stream, and from a graph replayed on new
    inputs with eager work in between."""
    rows, vocab = 20, 3000
    logits = rows_of(rows, vocab, F32, 1)
    values, indices, log_rest = make_record(rows, vocab, 9, 2)
    weights = torch.linspace(0.0, 1.0, rows, device=DEV)
    u = torch.rand(rows, device=DEV)

    def run():
        if op == "top":
            return tuple(top_logits(logits, 9))
        if op == "sample":
            return tuple(sample_tokens(logits, u, top_k=50, top_p=0.9)) + tuple(sample_tokens(logits, u, top_p=0.97))
        x = logits.detach().requires_grad_(True)
        loss = distillation_loss(x, values, indices, log_rest, weights=weights)
        return loss.detach(), torch.autograd.grad(loss, x, unit_gradient(loss))[0]

    want = run()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream(DEV).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for rep in range(3):
        logits.copy_(rows_of(rows, vocab, F32, 10 + rep))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        _ = torch.ones(64, device=DEV).sum().item()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), rep


def test_same_inputs_same_bits():
    logits = rows_of(50, 40001, BF16, 1)
    values, indices, log_rest = make_record(50, 40001, 20, 2)
    u = torch.rand(50, device=DEV)
    for run in (
        lambda: tuple(top_logits(logits, 100)),
        lambda: (distillation_loss(logits, values, indices, log_rest),),
        lambda: tuple(sample_tokens(logits, u, top_p=0.99)),
    ):
        first = run()
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_refusals():
    x = rows_of(3, 50, F32, 1)
    values, indices, log_rest = make_record(3, 50, 5, 2)
    u = torch.rand(3, device=DEV)
    with pytest.raises(ValueError, match="k <="):
        top_logits(x, 51)
    with pytest.raises(ValueError, match="temperature"):
        top_logits(x, 5, temperature=0.0)
    with pytest.raises(NotImplementedError, match="1024"):
        top_logits(torch.zeros(1, 2000, device=DEV), 1025)
    with pytest.raises(NotImplementedError, match="classes"):
        top_logits(torch.zeros(1, (1 << 20) + 1, device=DEV), 5)
    with pytest.raises(TypeError, match="logits"):
        top_logits(x.double(), 5)
    with pytest.raises(ValueError, match="values"):
        distillation_loss(x, values[:2], indices, log_rest)
    with pytest.raises(TypeError, match="indices"):
        distillation_loss(x, values, indices.int(), log_rest)
    with pytest.raises(ValueError, match="log_rest"):
        distillation_loss(x, values, indices, log_rest[:2])
    with pytest.raises(ValueError, match="weights"):
        distillation_loss(x, values, indices, weights=u.cpu())
    with pytest.raises(ValueError, match="reduction"):
        distillation_loss(x, values, indices, reduction="none")
    with pytest.raises(ValueError, match="temperature"):
        distillation_loss(x, values, indices, temperature=-1.0)
    with pytest.raises(NotImplementedError, match="lists"):
        distillation_loss(x, torch.zeros(3, 1025, device=DEV), torch.zeros(3, 1025, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="uniforms"):
        sample_tokens(x, u[:2])
    with pytest.raises(TypeError, match="uniforms"):
        sample_tokens(x, u.double())
    with pytest.raises(ValueError, match="top_p"):
        sample_tokens(x, u, top_p=0.0)
    with pytest.raises(ValueError, match="min_p"):
        sample_tokens(x, u, min_p=1.5)
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(x, u, temperature=math.nan)
    with pytest.raises(TypeError, match="top_k"):
        sample_tokens(x, u, top_k=torch.ones(3, device=DEV))
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(x, u, temperature=torch.ones(2, device=DEV))


def test_more_rows_than_one_grid_takes():
    """2^21 + 3 rows of three classes: launched in two grids, each row answered.
    Sums of 2^21 losses are f64 within and one f32 at the end: REL covers them."""
    rows, gen = (1 << 21) + 3, torch.Generator().manual_seed(77)
    x = torch.randn(rows, 3, generator=gen)
    teacher = torch.randn(rows, 3, generator=gen)
    got = top_logits(teacher.to(DEV), 3)
    _, indices = order_of(teacher)
    assert torch.equal(got.indices.cpu(), indices)
    drawn = sample_tokens(x.to(DEV), torch.zeros(rows, device=DEV), temperature=0.0)
    assert torch.equal(drawn.tokens.cpu(), order_of(x)[1][:, 0])
    logits = x.to(DEV).requires_grad_()
    loss = distillation_loss(logits, got.values, got.indices, reduction="sum")
    loss.backward()
    log_q, log_p = torch.log_softmax(x.double(), -1), torch.log_softmax(teacher.double(), -1)
    want = (log_p.exp() * (log_p - log_q)).sum()
    assert abs(float(loss.detach()) - float(want)) <= 4 * REL * float(want)
    assert float((logits.grad.cpu().double() - (log_q.exp() - log_p.exp())).abs().max()) <= REL


@pytest.mark.parametrize("levels", [3, 40, 700, 100000])
@pytest.mark.parametrize("vocab,k", [(700, 300), (5000, 257), (5000, 900), (40000, 1024)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_lists_of_more_and_fewer_equal_logits(levels, vocab, k, dtype):
    gen = torch.Generator().manual_seed(levels + vocab + k)
    x = (torch.randint(0, levels, (5, vocab), generator=gen).double() / levels * 12 - 4).to(dtype)
    x[3] = x[3].sort().values  # rising
    x[4] = x[4].sort(descending=True).values
    check_top(x.to(DEV), k)


@pytest.mark.parametrize("vocab", [7, 130, 5000, 40007])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_rows_answer_is_the_same_in_large_and_small_batches(vocab, dtype):
    """Batches of 700 rows and of 50 take different numbers of threads a row;
    lists and tokens are the same bits, log-masses within their bound."""
    x, u = rows_of(700, vocab, dtype, vocab), torch.rand(700, generator=torch.Generator().manual_seed(1)).to(DEV)
    part = slice(300, 350)
    k = min(vocab, 40)
    check_top(x, k)
    small, large = top_logits(x[part], k), top_logits(x, k)
    assert torch.equal(small.values, large.values[part]) and torch.equal(small.indices, large.indices[part])
    for kw in ({}, dict(top_p=0.9), dict(top_k=50, min_p=0.02), dict(top_k=300, top_p=0.95), dict(temperature=0.0),
               dict(temperature=3.0, top_p=0.6), dict(min_p=0.1)):
        small, large = sample_tokens(x[part], u[part], **kw), sample_tokens(x, u, **kw)
        assert torch.equal(small.tokens, large.tokens[part]), kw
        assert torch.equal(small.log_probs, large.log_probs[part]), kw


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", [
    "a new inner dimension", "inner dimension broadcast", "a new middle dimension", "two new dimensions",
    "outer dimension broadcast", "both broadcast", "slice", "one of the inner dimension", "every second row", "classes apart",
])
def test_distillation_leading_dimensions_and_layouts(layout, dtype):
    """Loss and gradient of logits in any layout are those of a contiguous copy."""
    base = rows_of(4 * 6, 500, dtype, 1, pad=4).unflatten(0, (4, 6))
    x = {
        "a new inner dimension": lambda: base[:, 0][:, None].expand(4, 8, 500),
        "inner dimension broadcast": lambda: base[:, :1].expand(4, 6, 500),
        "a new middle dimension": lambda: base[:, None].expand(4, 3, 6, 500),
        "two new dimensions": lambda: base[:, 0][:, None, None].expand(4, 2, 3, 500),
        "outer dimension broadcast": lambda: base[:1].expand(4, 6, 500),
        "both broadcast": lambda: base[:1, :1].expand(4, 6, 500),
        "slice": lambda: base[..., 3:450],
        "one of the inner dimension": lambda: base[:, 1],
        "every second row": lambda: base[:, ::2],
        "classes apart": lambda: base.transpose(1, 2).contiguous().transpose(1, 2),
    }[layout]()
    lead, vocab, k = x.shape[:-1], x.shape[-1], 7
    values, indices, log_rest = (t.reshape(*lead, *t.shape[1:]) for t in make_record(x.numel() // vocab, vocab, k, 2, t=1.5))
    weights = torch.linspace(0.0, 2.0, log_rest.numel(), device=DEV).reshape(lead)

    def run(logits):
        logits = logits.detach().requires_grad_(True)
        loss = distillation_loss(logits, values, indices, log_rest, weights=weights, temperature=1.5)
        loss.backward()
        with torch.no_grad():
            alone = distillation_loss(logits, values, indices, log_rest, weights=weights, temperature=1.5)
        return loss.detach(), alone, logits.grad

    assert all(torch.equal(a, b) for a, b in zip(run(x), run(x.contiguous())))
    check_distill(x.contiguous(), values, indices, log_rest, weights, t=1.5)


def distill_reference_by_rows(logits, values, indices, log_rest, weights, t=1.0):
    """distill_reference for many rows: the same formulas in 64 bits, a few
    hundred rows at a time, on the GPU. Loss, gradient and the bound of its
    error before it is stored, of the weighted mean."""
    rows, vocab = logits.shape
    w_all = torch.ones(rows, dtype=torch.float64, device=DEV) if weights is None else weights.double()
    total, loss, grads, bounds = w_all.sum(), 0.0, [], []
    for part in torch.arange(rows).split(max(1, (1 << 23) // vocab)):
        part = slice(int(part[0]), int(part[-1]) + 1)
        at, w = indices[part], w_all[part, None]
        here = at >= 0
        used = here.any(1, keepdim=True) & (w != 0)
        log_q = torch.log_softmax(logits[part].double() / t, 1)
        teacher = (values[part].double() / t).masked_fill(~here, -math.inf)
        if log_rest is not None:
            teacher = torch.cat((teacher, log_rest[part, None].double()), 1)
        log_p = torch.log_softmax(teacher, 1)
        p = log_p.exp()
        q, k = log_q.exp(), at.shape[1]
        spread = torch.zeros(len(at), vocab + 1, dtype=torch.float64, device=DEV)  # p by class; the last column: none
        spread.scatter_(1, torch.where(here, at, vocab), p[:, :k])
        listed = torch.zeros_like(spread, dtype=torch.bool).scatter_(1, torch.where(here, at, vocab), True)[:, :vocab]
        spread = torch.where(listed, spread[:, :vocab], 0.0)
        terms = torch.where(here & (p[:, :k] > 0), p[:, :k] * (log_p[:, :k] - log_q.gather(1, at.clamp(min=0))), 0.0).sum(1)
        ratio = torch.zeros(len(at), 1, dtype=torch.float64, device=DEV)
        if log_rest is not None:
            log_q0 = torch.logsumexp(log_q.masked_fill(listed, -math.inf), 1)
            p0 = p[:, k]
            terms += torch.where(p0 > 0, p0 * (log_p[:, k] - log_q0), 0.0)
            ratio = torch.where(p0 > 0, p0 / log_q0.exp(), 0.0)[:, None]
        loss += torch.where(used[:, 0], w[:, 0] * t * t * terms, 0.0).sum()
        coef = t * w / total
        g = torch.where(listed, q - spread, q * (1 - ratio))
        b = torch.where(listed, q + spread, q * (1 + ratio))
        grads.append(torch.where(used, coef * g, 0.0))
        bounds.append(torch.where(used, REL * coef * b, 0.0))
    return loss / total, torch.cat(grads), torch.cat(bounds)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("rows,vocab,k", [(4099, 300, 8), (4099, 5, 2), (700, 9000, 33)])
def test_distillation_scaled_losses(rows, vocab, k, rest, dtype):
    """A loss scaled against f16's underflow (a mean over thousands of rows has
    gradients below its smallest number): the gradient is the formula's times
    the scale, rounded once. A scale of one that the host does not know, and a
    second backward through the same graph, too."""
    logits = rows_of(rows, vocab, dtype, 3)
    values, indices, log_rest = make_record(rows, vocab, k, 4, t=2.0, rest=rest)
    weights = torch.rand(rows, generator=torch.Generator().manual_seed(5)).to(DEV)
    weights[::7] = 0.0
    want_loss, want, bound = distill_reference_by_rows(logits, values, indices, log_rest, weights, t=2.0)

    def check(grad, factor):
        off = (grad.double() - factor * want).abs() - (abs(factor) * bound + HALF_ULP[dtype] * (factor * want).abs() + SMALLEST[dtype])
        assert (off <= 0).all(), (factor, off.max())

    x = logits.detach().requires_grad_(True)
    for factor in (65536.0, -0.375, 1.0):
        loss = distillation_loss(x, values, indices, log_rest, weights=weights, temperature=2.0)
        assert abs(float(loss.detach()) - float(want_loss)) <= 4 * REL * (1 + abs(float(want_loss)))
        (first,) = torch.autograd.grad(factor * loss, x, retain_graph=True)
        check(first, factor)
        (second,) = torch.autograd.grad(loss, x, torch.tensor(2 * factor, device=DEV))
        check(second, 2 * factor)
        if factor == 1.0:
            again = distillation_loss(x, values, indices, log_rest, weights=weights, temperature=2.0)
            assert torch.equal(first, torch.autograd.grad(again, x, unit_gradient(again))[0])


def test_distillation_scaled_loss_in_a_graph():
    """The scaled 16-bit backward captured and replayed on new inputs."""
    logits = rows_of(600, 700, F16, 1)
    values, indices, log_rest = make_record(600, 700, 9, 2)
    factor = torch.tensor(1024.0, device=DEV)
    weights = torch.linspace(0.0, 1.0, 600, device=DEV)

    def run():
        x = logits.detach().requires_grad_(True)
        loss = distillation_loss(x, values, indices, log_rest, weights=weights)
        return torch.autograd.grad(loss, x, factor)[0]

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for rep in range(4):
        logits.copy_(rows_of(600, 700, F16, 10 + rep))
        factor.fill_((1024.0, 1.0, 0.5, 4096.0)[rep])
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        _ = torch.ones(64, device=DEV).sum().item()
        assert torch.equal(out, want), rep


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distillation_has_no_second_derivative(dtype):
    """With create_graph the gradient is the same, and whatever would need its
    derivative raises instead of leaving that part out."""
    values, indices, log_rest = make_record(4, 257, 6, 2)
    x = rows_of(4, 257, dtype, 1).requires_grad_(True)
    (want,) = torch.autograd.grad(distillation_loss(x, values, indices, log_rest), x)

    def loss_and_grad(**kw):
        loss = distillation_loss(x, values, indices, log_rest)
        return loss, torch.autograd.grad(loss, x, create_graph=True, **kw)[0]

    loss, grad = loss_and_grad()
    assert torch.equal(grad, want) and grad.requires_grad
    with pytest.raises(RuntimeError, match="differentiated once"):
        (loss + grad.float().square().sum()).backward()
    _, grad = loss_and_grad()
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(grad.float().square().sum(), x, allow_unused=True)
    incoming = torch.tensor(2.0, device=DEV, requires_grad=True)  # nor the derivative by the incoming gradient
    _, grad = loss_and_grad(grad_outputs=incoming)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(grad.float().sum(), incoming)
    # a graph that does not go through it
    distillation_loss(x, values, indices, log_rest).backward(create_graph=True)
    assert torch.equal(x.grad.detach(), want)
    x.grad = None


@pytest.mark.parametrize("requires_grad", [False, True])
def test_distillation_has_no_forward_mode_derivative(requires_grad):
    """A dual number is refused, where its tangent would be dropped; outside of
    the level the same logits are taken."""
    import torch.autograd.forward_ad as forward_ad

    values, indices, log_rest = make_record(4, 257, 6, 2)
    x = rows_of(4, 257, F32, 1).requires_grad_(requires_grad)
    want = distillation_loss(x, values, indices, log_rest).detach()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            distillation_loss(dual, values, indices, log_rest)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            distillation_loss(dual, values, indices, log_rest)
        assert torch.equal(distillation_loss(x, values, indices, log_rest).detach(), want)
        assert torch.equal(distillation_loss(dual.detach(), values, indices, log_rest), want)
    assert torch.equal(distillation_loss(x, values, indices, log_rest).detach(), want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [60, 1000, 33000, 100003])
def test_top_logits_nan_and_infinity_among_the_others(vocab, dtype):
    """More NaNs than the list holds beside infinities of either sign: the
    log-mass of the others is NaN; infinities alone make it infinite."""
    x = rows_of(6, vocab, dtype, 3)
    for r, (nans, inf) in enumerate(((15, math.inf), (15, -math.inf), (5, math.inf), (4, math.inf), (0, math.inf), (15, 0.0))):
        x[r, vocab // 3 : vocab // 3 + nans] = math.nan
        x[r, [1, vocab - 2]] = inf
    x[5, :] = torch.where(torch.isnan(x[5]), x[5], -math.inf)
    for k in (1, 4, 14):
        check_top(x, k)
        check_top(x, k, temperature=0.3)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_distillation_gradient_is_rounded_once_far_from_zero(dtype):
    """The teacher's list lies 2^80 below the student's other logits, around
    2^190: the constants of the gradient's exponents are at their largest.
    In f32, an exponent off by e moves a gradient by e ln 2 of itself. A constant
    below 2^8 is off by 2^-17 at most, a log-sum below 2^7 by 2^-18, half an ulp
    each, the instruction and the row's factor by 4 u: 1e-5 of a gradient, beside
    the half ulp of the type's own rounding. A constant above 2^8 would be off by
    2^-16."""
    rows, vocab, k = 20000, 64, 3
    gen = torch.Generator().manual_seed(7)
    x = 180.0 + 6.0 * torch.rand(rows, vocab, generator=gen)
    indices = torch.rand(rows, vocab, generator=gen).argsort(1)[:, :k].contiguous()
    x.scatter_(1, indices, 131.0 - 3.0 * torch.rand(rows, k, generator=gen))
    logits = x.to(dtype).to(DEV).requires_grad_(True)
    values = torch.zeros(rows, k, device=DEV)
    distillation_loss(logits, values, indices.to(DEV), reduction="sum").backward()
    want = torch.softmax(logits.detach().double(), 1)  # of a class outside the list
    near_zero = 2.0**-13  # above f16's subnormal numbers
    mantissa, exponent = torch.frexp(want)
    half_ulp = torch.ldexp(torch.ones_like(mantissa), exponent - (12 if dtype == F16 else 9))
    off = ((logits.grad.double() - want).abs() - half_ulp) / want
    off.scatter_(1, indices.to(DEV), 0.0)
    assert (want > near_zero).double().mean() > 0.5
    assert off[want > near_zero].max() <= 1e-5


def test_sample_top_k_of_any_int64():
    """0 and less are no limit, however far below; more than the classes is all."""
    logits = rows_of(8, 700, F32, 2)
    u = torch.full((8,), 0.97, device=DEV)
    top_k = torch.tensor([0, -1, -(2**31) - 5, 5 - 2**32, -(2**63), 2**31 + 1, 2**63 - 1, 3], device=DEV)
    got, want = sample_tokens(logits, u, top_k=top_k), sample_tokens(logits, u)
    assert torch.equal(got.tokens[:7], want.tokens[:7]) and torch.equal(got.log_probs[:7], want.log_probs[:7])
    assert int(got.tokens[7]) in order_of(logits[7].cpu())[1][:3].tolist()


@pytest.mark.parametrize("rest,weighted", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize(
    "rows,vocab,k,dtype,grid",
    [  # one more row than the workgroups, or several for each; the numbers of threads and of pieces a thread
        (4099, 10, 4, F32, 4096),
        (9001, 40, 9, F32, 4096),
        (9001, 700, 130, F32, 4096),
        (8500, 3101, 70, BF16, 4096),
        (3300, 5003, 33, BF16, 1536),
        (3300, 5003, 17, F32, 1536),
        (1301, 20000, 64, F16, 512),
        (1301, 20003, 5, F32, 512),
        (700, 70003, 300, BF16, 256),
    ],
)
def test_distillation_several_rows_a_workgroup(rows, vocab, k, dtype, grid, rest, weighted):
    """More rows than workgroups that hold them (`grid`): every one has its next
    row's list and pieces under way, rows of weight 0 and without a list in
    between, first, last and alone."""
    gen = torch.Generator().manual_seed(rows + k)
    logits = rows_of(rows, vocab, dtype, rows, pad=1)
    teacher = torch.randn(rows, vocab, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV) * 3
    values, indices = torch.sort(teacher, dim=1, descending=True, stable=True)
    log_rest = torch.logsumexp(values[:, k:].double(), 1).float() if rest else None
    values, indices = values[:, :k].to(dtype), indices[:, :k].clone()
    length = torch.where(torch.rand(rows, generator=gen) < 0.5, k, torch.randint(1, k + 1, (rows,), generator=gen))
    for empty in (slice(3, 5), slice(11, None, grid), slice(grid + 1, grid + 3), slice(rows - 2, rows - 1)):
        length[empty] = 0
    far = [r for r in (6, grid, grid + 6, 2 * grid + 6) if r < rows]  # their sums leave the unit of the list's largest
    length[far] = k
    for r in far:
        listed = logits[r].gather(0, indices[r])
        logits[r] += 200.0
        logits[r].scatter_(0, indices[r], listed)
    indices[torch.arange(k, device=DEV) >= length.to(DEV)[:, None]] = -1
    weights = None
    if weighted:
        weights = torch.where(torch.rand(rows, generator=gen) < 0.3, 0.0, 0.5 + torch.rand(rows, generator=gen))
        for out in (slice(0, 3), slice(7, None, grid), slice(grid, grid + 2), slice(rows - 1, rows)):
            weights[out] = 0.0
        weights[5] = 1.0
        weights[far] = 1.0
        weights = weights.to(DEV)
    want_loss, want, bound = distill_reference_by_rows(logits, values, indices, log_rest, weights)

    def run():
        x = logits.detach().requires_grad_(True)
        loss = distillation_loss(x, values, indices, log_rest, weights=weights)
        loss.backward()
        return loss.detach(), x.grad

    loss, grad = run()
    assert abs(float(loss) - float(want_loss)) <= 2 * REL * (1 + abs(float(want_loss)))
    for part in torch.arange(rows).split(max(1, (1 << 23) // vocab)):
        part = slice(int(part[0]), int(part[-1]) + 1)
        off = (grad[part].double() - want[part]).abs() - (bound[part] + HALF_ULP[dtype] * want[part].abs() + SMALLEST[dtype])
        assert (off <= 0).all(), (part, off.max(), torch.nonzero((off > 0).any(1))[:5])
    nothing = length.to(DEV) == 0
    if weighted:
        nothing |= weights == 0
    assert not grad[nothing].any()
    again = run()
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)


MOST = 1 << 20  # classes: the limit


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,shift", [(2, 1024, 0), (3, 5, 1), (1, 300, 3)])
def test_top_logits_of_the_most_classes(rows, k, shift, dtype):
    check_top(rows_of(rows, MOST, dtype, k, shift=shift), k, temperature=1.3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("vocab,k", [(MOST, 64), (MOST, 1024), (MOST - 3, 7), (516097, 20), (516096, 20), (516000, 20), (515000, 20)])
def test_distillation_of_the_most_classes(vocab, k, rest, dtype):
    """The limit, and around the vocabulary whose bitmap takes 64 KB of LDS. A
    thread's run of a sum is 256 pieces at most, 2e-5 as for the sizes above."""
    logits = rows_of(3, vocab, dtype, k)
    values, indices, log_rest = make_record(3, vocab, k, 3, rest=rest, values_dtype=dtype)
    indices[1, k // 2 :] = -1
    indices[0, 0] = vocab - 1 if not (indices[0] == vocab - 1).any() else indices[0, 0]
    check_distill(logits, values, indices, log_rest, torch.tensor([1.0, 2.0, 0.5], device=DEV))


def sample_reference_wide(x, u, top_k=0, top_p=1.0, min_p=0.0):
    """sample_reference for wide rows: whole logits [rows, vocab] (int64; hidden
    ones far below), in whole numbers."""
    m = x.amax(1, keepdim=True)
    w = torch.where(m - x < 63, ONE >> (m - x).clamp(max=62), 0)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    kept = w.gather(1, order)
    if top_k > 0:
        kept[:, top_k:] = 0
    before = kept.cumsum(1) - kept
    if top_p < 1.0:
        total = kept.sum(1, keepdim=True).double()
        limit = (float(torch.tensor(top_p, dtype=F32)) * total).to(torch.int64).clamp(min=1)
        kept = torch.where(before < limit, kept, 0)
    kept = torch.where(kept.double() >= float(torch.tensor(min_p, dtype=F32)) * ONE, kept, 0)
    by_index = torch.zeros_like(w).scatter(1, order, kept)
    running = by_index.cumsum(1)
    total = running[:, -1:]
    target = torch.minimum((u.double()[:, None] * total.double()).to(torch.int64), total - 1)
    token = (running <= target).sum(1, keepdim=True)
    return token[:, 0], (by_index.gather(1, token).double() / total.double()).log()[:, 0]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-6, -30])
def test_sample_of_the_most_classes(low, dtype):
    gen = torch.Generator().manual_seed(-low)
    rows = 3
    x = torch.randint(low, 1, (rows, MOST), generator=gen)
    x[2] = -(torch.arange(MOST) % 97) - 1
    x[2, MOST - 1] = 0  # the last class alone is the largest
    x[:, 5:100] = -(1 << 20)  # masked
    logits = torch.where(x < -1000, -math.inf, x.float()).to(dtype).to(DEV)
    for n, kw in enumerate((dict(), dict(top_k=50), dict(top_k=1000, top_p=0.9), dict(top_k=5000), dict(top_p=0.9),
                            dict(top_p=0.3, min_p=0.01), dict(min_p=0.2), dict(top_k=300000, top_p=0.5))):
        u = torch.rand(rows, generator=gen)
        u[0] = (0.0, 1.0 - 2.0**-24, 0.5)[n % 3]
        got = sample_tokens(logits, u.to(DEV), temperature=LOG2E, **kw)
        token, log_prob = sample_reference_wide(x, u, **kw)
        assert torch.equal(got.tokens.cpu(), token), kw
        assert torch.allclose(got.log_probs.cpu().double(), log_prob, rtol=1e-6, atol=1e-6), kw
    cold = sample_tokens(logits, torch.zeros(rows, device=DEV), temperature=0.0)
    assert torch.equal(cold.tokens.cpu(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, 0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [77, 3001, 50001])
@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_p=0.5), dict(top_p=0.7, min_p=0.001), dict(min_p=0.05),
                                dict(top_k=200, top_p=0.8), dict(top_k=25, top_p=0.95, min_p=0.01)])
def test_sample_against_64_bits_with_wide_gaps(vocab, dtype, kw):
    """As test_sample_against_64_bits, of rows whose cuts lie in wide gaps: 30
    raised classes hold nearly all of the mass, a hundredth of it and more each,
    and the others weigh a millionth of the largest, so that the cut is among the
    raised ones and hardly ever within 1e-4 of the limit."""
    rows, t = 200, 0.8
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=gen) * 0.5 - 12.0
    raised = torch.rand(rows, vocab, generator=gen).argsort(1)[:, :30]
    x.scatter_(1, raised, torch.rand(rows, 30, generator=gen))
    logits = x.to(dtype).to(DEV)
    u = torch.rand(rows, generator=gen)
    got = sample_tokens(logits, u.to(DEV), temperature=t, **kw)
    values, order = order_of(logits.cpu())
    w = torch.exp((values - values[:, :1]) / t)
    top_k, top_p, min_p = kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0)
    if top_k > 0:
        w[:, top_k:] = 0.0
    before = w.cumsum(1) - w
    limit = top_p * w.sum(1, keepdim=True)
    near = ((before - limit).abs() < 1e-4 * limit).any(1) & (top_p < 1)
    near |= ((w - min_p).abs() < 1e-5).any(1) & (min_p > 0)
    kept = w >= min_p
    if top_p < 1:
        kept &= before < limit
    w = torch.where(kept, w, 0.0)
    by_index = torch.zeros_like(w).scatter(1, order, w)
    by_index /= by_index.sum(1, keepdim=True)
    upto = by_index.cumsum(1)
    token = got.tokens.cpu()[:, None]
    p, high, ok = by_index.gather(1, token)[:, 0], upto.gather(1, token)[:, 0], ~near
    assert ok.sum() >= 0.95 * rows
    assert (p[ok] > 0).all()
    assert ((u.double() <= high + 3e-5) & (u.double() >= high - p - 3e-5))[ok].all()
    assert torch.allclose(got.log_probs.cpu().double()[ok], p[ok].log(), rtol=REL, atol=REL)


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_distillation_backward_captured_apart_from_its_forward(dtype, weighted):
    """A backward in a graph of its own writes its gradient in every replay,
    whatever the factor and whatever became of the last one; one that its
    forward's graph holds too does so as well."""
    rows, vocab = 70, 900
    logits = rows_of(rows, vocab, dtype, 1)
    values, indices, log_rest = make_record(rows, vocab, 9, 2)
    weights = torch.linspace(0.0, 2.0, rows, device=DEV) if weighted else None
    factor = torch.ones((), device=DEV)

    def forward(x):
        return distillation_loss(x, values, indices, log_rest, weights=weights)

    def eager(by):
        x = logits.detach().requires_grad_(True)
        return torch.autograd.grad(forward(x), x, torch.full((), by, device=DEV))[0]

    eager(1.0)
    first, second, both = (torch.cuda.CUDAGraph() for _ in range(3))
    side = torch.cuda.Stream(DEV)
    x = logits.detach().requires_grad_(True)
    with torch.cuda.graph(first, stream=side):
        loss = forward(x)
    with torch.cuda.graph(second, pool=first.pool(), stream=side):
        (grad,) = torch.autograd.grad(loss, x, factor)
    y = logits.detach().requires_grad_(True)
    with torch.cuda.graph(both, stream=side):
        (together,) = torch.autograd.grad(forward(y), y, factor)
    # computed again or scaled where it was written: a rounding apart
    close = dict(rtol=4 * HALF_ULP[dtype], atol=2 * SMALLEST[dtype])
    for rep in range(2):
        logits.copy_(rows_of(rows, vocab, dtype, 20 + rep))
        first.replay()
        for by in (1.0, 0.5, 1.0, -2.0):
            factor.fill_(by)
            second.replay()
            both.replay()
            want = eager(by).float()
            assert torch.allclose(grad.float(), want, **close) and torch.allclose(together.float(), want, **close), (rep, by)
            grad.mul_(3.0)
            together.mul_(3.0)
