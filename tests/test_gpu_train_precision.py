"""The precision that the token losses keep: log-probabilities to a few 2^-24 before
any rounding of themselves, and losses formed from those. test_gpu_train.py allows
for f32 sums of whole runs; here the bounds are those of the arithmetic there is.

With u = 2^-24, p the classes' probabilities and a_i = log2(p_i / the largest):
  a term 2^a     the instruction has one unit in the last place, 2 u, perhaps on one
                 side for all terms; two roundings of the exponent, 2 ln 2 |a| u, and
                 four of the sum of sixteen terms, 4 u, independent of the others'.
                 Their sum, over the mass, is at most sum p_i (2 ln 2 |a_i| + 4) u, and
                 in all but a 1e-8 of the rows 6 sqrt(sum p_i^2 (2 ln 2 |a_i| + 4)^2 / 3) u
  the token's    exp of a f64 number by an f32 instruction: 2.5 u of it
  the logarithm  of a number from 0.7 to 1.5, at most 0.41, by an f32 function: two
                 units in the last place, u; 4 u of it where it is smaller
What follows is f64. A ratio is 2.5 u off by its own exponential."""
from __future__ import annotations

import math

import pytest
import torch

from tropnn_amd import policy_loss, preference_loss
from tropnn_amd.backends import train_hip as th
from tropnn_amd.backends.logits_hip import LOGITS_DTYPES

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
U = 2.0**-24


def rows_of(rows, vocab, dtype, seed, low=0.0):
    """Logits of N(0, 1), and a token for each row, its logit lowered by `low`."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=gen, device=DEV)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    logits.scatter_add_(1, tokens[:, None], torch.full((rows, 1), -low, device=DEV))
    return logits.to(dtype), tokens


def reference(logits, tokens, t=1.0):
    """(log-probabilities, their bounds) in 64 bits."""
    z = logits.double() / t
    at = tokens[:, None]
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    others = p.scatter(1, at, 0.0)
    mass = others.sum(1)
    a = (z - z.amax(1, keepdim=True)).abs() / math.log(2.0)
    each = others * (2 * math.log(2.0) * a + 4)
    independent = each.sum(1)
    if logits.dtype == F32:  # equal logits, of which 16 bits have many, are rounded alike
        independent = torch.minimum(independent, 6 * (each.square().sum(1) / 3).sqrt())
    lp = log_p.gather(1, at)[:, 0]
    lp = torch.where(mass < 0.5, torch.log1p(-mass), lp)
    return lp, U * (2 * mass + independent + 2.5 * (1 - mass) * mass + torch.minimum(4 * lp.abs(), torch.ones_like(lp)))


def exact_log_probs(logits, tokens, t=1.0):
    """What the C ABI gives without the last rounding."""
    out = torch.empty(len(tokens), dtype=F64, device=DEV)
    rc = th.load_train_library().tropnn_hip_token_log_probs(
        *logits.shape, logits.stride(0), logits.data_ptr(), LOGITS_DTYPES[logits.dtype], tokens.data_ptr(), t, None, out.data_ptr(),
        None, torch.cuda.current_stream(DEV).cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,low,t", [
    (3000, 3, 0.0, 1.0), (2000, 9, 0.0, 0.7), (2000, 9, -12.0, 1.0), (1100, 700, 0.0, 1.0), (1100, 700, 8.0, 1.6), (300, 9001, -14.0, 1.0),
    (300, 40003, 8.0, 1.0), (40, 131072, 0.0, 1.0), (40, 131072, 8.0, 1.3), (9, 1 << 20, 4.0, 1.0),
])
def test_log_probs_before_their_rounding(rows, vocab, low, t, dtype):
    logits, tokens = rows_of(rows, vocab, dtype, vocab + int(low), low)
    want, bound = reference(logits, tokens, t)
    got = exact_log_probs(logits, tokens, t)
    off = (got - want).abs() - bound
    assert (off <= 0).all(), (float((got - want).abs().max()) / U, float(off.max()) / U)


PAIRS = 24
FORMS = [(64, 131072), (300, 40003)]  # read for the loss alone, and held on chip for the gradient too


@pytest.mark.parametrize("rows,vocab", FORMS)
def test_a_policy_loss_that_is_the_rest_of_its_terms(rows, vocab):
    """Two rows whose terms are alike but for a thousandth and of both signs, at
    log-probabilities near -20, whose rounding to f32 would be off by up to 16 u."""
    logits, tokens = rows_of(rows, vocab, F32, rows, 8.5)
    lp, bound = reference(logits, tokens)
    old = lp.float()  # exact as given, whatever it was rounded from
    advantages = torch.ones(rows, device=DEV)
    advantages[1::2] = -0.999
    ratio = torch.exp(lp - old.double())
    caught = 0
    for k in range(PAIRS):
        pair = [2 * k, 2 * k + 1]
        weights = torch.zeros(rows, device=DEV)
        weights[pair] = 1.0
        x = logits.detach().requires_grad_(True)
        got = policy_loss(x, tokens, old, advantages, weights=weights).loss.item()
        terms = -(ratio * advantages.double())[pair] / 2
        want = float(terms.sum())
        allowed = float((terms.abs() * (bound[pair] + 2.5 * U)).sum()) + U * abs(want)
        assert 2e-4 < abs(want) < 1e-3 and abs(got - want) <= allowed, (k, got - want, allowed)
        # a loss from log-probabilities in f32 would not pass
        other = float(-advantages.double()[pair].sum() / 2)  # their ratios are one
        caught += abs(other - want) > allowed
    assert caught >= 2


@pytest.mark.parametrize("rows,vocab", FORMS)
def test_a_preference_loss_from_unrounded_sums(rows, vocab):
    """A pair's loss by its log-probabilities near -20: half of their errors."""
    logits, tokens = rows_of(rows, vocab, F32, rows + 1, 8.5)
    lp, bound = reference(logits, tokens)
    half = rows // 2
    known = lp.float().view(2, half)
    h = (lp.view(2, half) - known.double()).diff(dim=0)[0].neg()
    caught = 0
    for k in range(PAIRS):
        weights = torch.zeros(half, device=DEV)
        weights[k] = 1.0
        got = preference_loss(logits.view(2, half, 1, vocab), tokens.view(2, half, 1), known, beta=1.0, margin=-3.0, weights=weights)
        want = math.log1p(math.exp(-float(h[k]) - 3.0))
        slope = 1 / (1 + math.exp(3.0))
        allowed = slope * float(bound.view(2, half)[:, k].sum()) + U * want
        assert abs(got.loss.item() - want) <= allowed, (k, got.loss.item() - want, allowed)
        caught += abs(math.log1p(math.exp(-3.0)) - want) > allowed  # sums in f32 would be the reference's own
    assert caught >= 2
