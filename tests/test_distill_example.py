"""The distillation example's host side, without a GPU."""
from __future__ import annotations

import math

import torch

from tropnn_amd import SampledTokens
from tropnn_amd.examples import distill


def test_a_row_without_an_answer_does_not_index_with_it(monkeypatch):
    """sample_tokens answers -1 for logits with a NaN. That is what generate
    returns for the row, and no class for a model to look up."""
    seen = []

    def model(window):
        seen.append(window.clone())
        return torch.zeros(len(window), 9)

    def drawn(logits, uniforms, **kw):
        return SampledTokens(torch.tensor([-1, 5, -1]), torch.tensor([math.nan, -0.5, math.nan]))

    monkeypatch.setattr(distill, "sample_tokens", drawn)
    tokens, log_probs = distill.generate(model, torch.tensor([[1, 2], [3, 4], [7, 8]]), 3)
    assert tokens.tolist() == [[-1] * 3, [5] * 3, [-1] * 3]
    assert torch.isnan(log_probs[[0, 2]]).all() and (log_probs[1] == -0.5).all()
    for window in seen:
        assert int(window.min()) >= 0
    assert seen[1].tolist() == [[2, 0], [4, 5], [8, 0]]


def test_an_epochs_loss_is_the_mean_over_its_contexts(monkeypatch):
    """Whatever batches they come in: a last one that is shorter, or one alone."""

    def step(model, optimizer, contexts, rec, *, temperature):
        return contexts.double().sum(1).mean()

    monkeypatch.setattr(distill, "distill_step", step)
    monkeypatch.setattr(distill, "FusedAdam", lambda *a, **kw: None)
    monkeypatch.setattr(distill, "record", lambda teacher, contexts, k, temperature: [contexts])
    monkeypatch.setattr(distill, "TopLogits", lambda *t: t)
    monkeypatch.setattr(distill, "generate", lambda *a, **kw: None)
    for contexts, batch in ((10, 4), (3, 512), (8, 4)):
        out = distill.run(vocab=50, contexts=contexts, batch=batch, epochs=1, device="cpu")
        want = distill.make_contexts(contexts, 50).double().sum(1).mean()
        assert abs(out["losses"][0] - float(want)) <= 1e-5 * float(want)
