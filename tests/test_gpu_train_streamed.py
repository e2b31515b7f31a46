"""The token losses on logits past the caches: more than 256 MB of them, where every
kernel takes its non-temporal form (scores from 128 MB on, with a gradient to come
from 256 MB; gradients and rows held on chip from 128 MB on). Odd vocabularies, so
that 16-bit rows start on and off 4-byte boundaries, with tokens in the loose logits
before and behind the 16-byte pieces. Bounds as in test_gpu_train.py."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_train import (BF16, DEV, F16, F32, F64, U, check, check_policy, policy_inputs, reference_gradient, reference_policy,
                            reference_rows)
from tropnn_amd import policy_loss, preference_loss, token_log_probs

pytestmark = pytest.mark.gpu
SIZES = [(F32, 1100, 65531, 1), (F16, 1100, 131067, 2), (BF16, 1100, 131067, 0)]  # type, rows, vocab, columns between rows


def inputs(dtype, rows, vocab, pad):
    gen = torch.Generator(device=DEV).manual_seed(vocab + pad)
    wide = torch.full((rows, vocab + pad), math.nan, dtype=dtype, device=DEV)
    logits = wide[:, :vocab]
    logits.copy_(3 * torch.randn(rows, vocab, generator=gen, device=DEV))
    assert logits.numel() * logits.element_size() > 1 << 28
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    ends = torch.cat([torch.arange(10), vocab - 1 - torch.arange(10), vocab // 2 + torch.arange(10)]).to(DEV)
    tokens[:60] = ends.repeat_interleave(2)  # each on an even and an odd row
    tokens[70::5] = -1
    return logits, tokens


@pytest.mark.parametrize("dtype,rows,vocab,pad", SIZES)
def test_log_probs(dtype, rows, vocab, pad):
    logits, tokens = inputs(dtype, rows, vocab, pad)
    lp, bound, _, _ = reference_rows(logits, tokens, 1.1)
    with torch.no_grad():
        check(token_log_probs(logits, tokens, temperature=1.1), lp, bound, "log_probs alone")
    x = logits.detach().requires_grad_(True)
    got = token_log_probs(x, tokens, temperature=1.1)
    check(got, lp, bound, "log_probs")
    by = torch.randn(rows, generator=torch.Generator().manual_seed(1))
    by[5] = 0.0
    got.backward(by.to(DEV))
    want, grad_bound = reference_gradient(logits, tokens, 1.1, by.double(), torch.zeros(rows, dtype=F64))
    check(x.grad, want, grad_bound, "grad")


@pytest.mark.parametrize("dtype,rows,vocab,pad", SIZES)
def test_policy(dtype, rows, vocab, pad):
    logits, tokens = inputs(dtype, rows, vocab, pad)
    old, advantages, refs, weights = policy_inputs(logits, tokens, 1.0, 8, low=0.2, high=0.2, weighted=True)
    weights[:60] = 1.0
    check_policy(logits, tokens, old, advantages, refs, weights)
    check_policy(logits, tokens, old, advantages, None, None, scale=1024.0)
    want = reference_policy(logits, tokens, old, advantages, refs, weights, 1.0, 0.2, 0.2, 0.1, 1024.0, True)
    x = logits.detach().requires_grad_(True)
    (policy_loss(x, tokens, old, advantages, refs, weights=weights).loss * 1024.0).backward()
    check(x.grad, want[4], want[5], "another incoming gradient")


@pytest.mark.parametrize("dtype,rows,vocab,pad", SIZES)
def test_preference(dtype, rows, vocab, pad):
    logits, tokens = inputs(dtype, rows, vocab, pad)
    pairs = logits.as_strided((2, 10, 55, vocab), (550 * (vocab + pad), 55 * (vocab + pad), vocab + pad, 1))
    tokens = tokens.view(2, 10, 55)
    lp, bound, _, _ = reference_rows(logits, tokens, 1.0)
    sums, off = (torch.where(tokens >= 0, v.view(tokens.shape), 0.0).sum(2) for v in (lp, bound))
    noise = torch.randn(2, 10, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    reference = (sums + 3 * noise).float()
    x = pairs.detach().requires_grad_(True)
    got = preference_loss(x, tokens, reference)
    check(got.log_probs, sums, off + 2 * U * sums.abs(), "log_probs")
    h = 0.1 * (sums - reference.double()).diff(dim=0)[0].neg()
    h_off = 0.1 * off.sum(0)
    loss = torch.nn.functional.softplus(-h)
    check(got.loss, loss.mean(), (h_off + 8 * U * (1 + h.abs())).mean(), "loss")
    got.loss.backward()
    by, by_off = -0.1 * torch.sigmoid(-h) / 10, (0.1 * 0.25 * h_off + 8 * U * 0.1) / 10
    by, by_off = (torch.stack(v)[:, :, None].expand(2, 10, 55).reshape(-1) for v in ((by, -by), (by_off, by_off)))
    want, grad_bound = reference_gradient(logits, tokens.reshape(-1), 1.0, by, by_off)
    check(x.grad.view(rows, vocab), want, grad_bound, "grad")
