"""The distillation example end to end: record, training, answers."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from tropnn_amd import FusedAdam, TopLogits
from tropnn_amd.examples.distill import (
    PairwiseTokenModel,
    TableTeacher,
    distill_step,
    generate,
    make_contexts,
    record,
    run,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_run_learns_and_answers():
    out = run(vocab=257, contexts=2048, batch=256, k=16, epochs=4)
    losses = out["losses"]
    assert all(math.isfinite(v) and v >= 0 for v in losses)
    assert losses[-1] < 0.9 * losses[0], losses
    for name in ("teacher", "student"):
        tokens, log_probs = out[name]
        assert tokens.shape == log_probs.shape == (8, 12) and tokens.dtype == torch.int64
        assert bool(((tokens >= 0) & (tokens < 257)).all())
        assert bool((log_probs <= 0).all()) and bool(torch.isfinite(log_probs).all())


def test_step_from_a_whole_record_is_the_soft_cross_entropys():
    """A record of every class leaves nothing to the rest: the step's loss is
    the divergence of the two softmaxes, and so are the gradients of the layers
    below the logits (f32 logits of order 1: 1e-4 relative to the largest)."""
    vocab = 129
    teacher = TableTeacher(vocab, seed=3).to(DEV)
    contexts = make_contexts(64, vocab, seed=4).to(DEV)
    rec = record(teacher, contexts, vocab, temperature=2.0)
    assert bool((rec.log_rest == -math.inf).all())

    grads = []
    for own in (True, False):
        model = PairwiseTokenModel(vocab, seed=5).to(DEV)
        if own:
            loss = distill_step(model, FusedAdam(model.parameters(), lr=0.0), contexts, rec, temperature=2.0)
        else:
            logq = F.log_softmax(model(contexts) / 2.0, -1)
            logp = F.log_softmax(teacher(contexts) / 2.0, -1)
            loss = 4.0 * F.kl_div(logq, logp, reduction="batchmean", log_target=True)
            loss.backward()
        grads.append((loss.detach(), [p.grad.clone() for p in model.parameters() if p.grad is not None]))
    (loss, got), (want_loss, want) = grads
    assert torch.allclose(loss, want_loss, rtol=1e-4, atol=1e-5)
    assert len(got) == len(want) > 2
    for g, w in zip(got, want):
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max())


def test_a_batch_of_a_record_is_the_batchs_record():
    teacher = TableTeacher(300, seed=1).to(DEV)
    contexts = make_contexts(40, 300, seed=2).to(DEV)
    whole = record(teacher, contexts, 12)
    part = record(teacher, contexts[8:24], 12)
    for a, b in zip(TopLogits(*(t[8:24] for t in whole)), part):
        assert torch.equal(a, b)


def test_generate_repeats_with_its_generator_and_greedy_takes_the_first():
    teacher = TableTeacher(211, seed=7).to(DEV)
    contexts = make_contexts(5, 211, seed=8).to(DEV)
    runs = [generate(teacher, contexts, 6, generator=torch.Generator(device=DEV).manual_seed(9), top_k=20) for _ in range(2)]
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    tokens, log_probs = generate(teacher, contexts, 3, temperature=0.0)
    window = contexts
    for step in range(3):
        first = teacher(window).argmax(-1)
        assert torch.equal(tokens[:, step], first)
        window = torch.cat([window, first.unsqueeze(1)], 1)[:, -2:]
    assert bool((log_probs == 0).all())
