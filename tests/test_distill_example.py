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
