"""A small token model of PairwiseLinear layers that learns from a stronger one
and then answers: the operators on rows of logits, used together.

The teacher is any function from contexts (token ids [batch, context]) to logits
[batch, vocab]. Its answer to a set of contexts is recorded once (`record`: the
k first logits and the log-mass of the others, k * 12 bytes a context instead
of vocab * 4), and the student trains on the record (`distill_step`), whose
batches need the teacher no more. `generate` draws tokens from either.

The training step is the one of the reference's loop (examples/emnist.py:218-224)
with the divergence from the record in the place of cross entropy.
"""
from __future__ import annotations

from typing import Callable

import torch
import torch.nn as nn
from torch import Tensor

from ..layers import PairwiseLinear
from ..logits import TopLogits, distillation_loss, sample_tokens, top_logits
from ..losses import unit_gradient
from ..optim import FusedAdam


class PairwiseTokenModel(nn.Module):
    """The next token's logits from the last `context` tokens: their embeddings
    side by side, then PairwiseLinear layers with no activation in between."""

    def __init__(self, vocab: int, *, context: int = 2, width: int = 32, hidden_dim: int = 128, tables: int = 64,
                 comparisons: int = 6, seed: int = 0) -> None:
        super().__init__()
        self.context = context
        self.embedding = nn.Embedding(vocab, width)
        with torch.no_grad():
            self.embedding.weight.normal_(generator=torch.Generator().manual_seed(seed))
        self.layers = nn.ModuleList([
            PairwiseLinear(context * width, hidden_dim, tables=tables, comparisons=comparisons, seed=seed),
            PairwiseLinear(hidden_dim, vocab, tables=tables, comparisons=comparisons, seed=seed + 1, input_grad="fused"),
        ])

    def forward(self, contexts: Tensor) -> Tensor:
        x = self.embedding(contexts).flatten(-2).unsqueeze(1)
        for layer in self.layers:
            x = layer(x)
        return x.squeeze(1)


class TableTeacher(nn.Module):
    """A teacher to learn from without a dataset: logits of the next token as a
    sum of one table row per context token, drawn from `seed`."""

    def __init__(self, vocab: int, *, context: int = 2, sharpness: float = 3.0, seed: int = 0) -> None:
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        self.context = context
        self.register_buffer("tables", torch.randn(context, vocab, vocab, generator=gen) * (sharpness / context**0.5))

    def forward(self, contexts: Tensor) -> Tensor:
        return sum(self.tables[i][contexts[:, i]] for i in range(self.context))


def make_contexts(count: int, vocab: int, context: int = 2, seed: int = 0) -> Tensor:
    return torch.randint(0, vocab, (count, context), generator=torch.Generator().manual_seed(seed))


@torch.no_grad()
def record(teacher: Callable[[Tensor], Tensor], contexts: Tensor, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The teacher's record for these contexts, at the temperature that it will
    be distilled at."""
    return top_logits(teacher(contexts), k, temperature=temperature)


def distill_step(model: nn.Module, optimizer: torch.optim.Optimizer, contexts: Tensor, rec: TopLogits, *,
                 temperature: float = 1.0, weights: Tensor | None = None) -> Tensor:
    """One training step on a batch of the record; returns the loss tensor. The
    backward starts from the kept unit gradient, so the loss's gradient is used
    as its launch wrote it."""
    optimizer.zero_grad(set_to_none=True)
    loss = distillation_loss(model(contexts), *rec, weights=weights, temperature=temperature)
    loss.backward(unit_gradient(loss))
    optimizer.step()
    return loss


@torch.no_grad()
def generate(model: Callable[[Tensor], Tensor], contexts: Tensor, steps: int, *, generator: torch.Generator | None = None,
             **sampling) -> tuple[Tensor, Tensor]:
    """`steps` tokens after each context and their log-probabilities, [batch,
    steps] both. The random numbers come from `generator`, one per token;
    `sampling` is sample_tokens' temperature, top_k, top_p and min_p. A token of
    -1 (logits with a NaN: no answer) is followed as if it were class 0."""
    batch, context = contexts.shape
    uniforms = torch.rand(steps, batch, generator=generator, device=contexts.device)
    tokens, log_probs = [], []
    window = contexts
    for step in range(steps):
        drawn = sample_tokens(model(window), uniforms[step], **sampling)
        tokens.append(drawn.tokens)
        log_probs.append(drawn.log_probs)
        window = torch.cat([window, drawn.tokens.clamp(min=0).unsqueeze(1)], 1)[:, -context:]
    return torch.stack(tokens, 1), torch.stack(log_probs, 1)


def run(*, vocab: int = 512, contexts: int = 8192, batch: int = 512, k: int = 32, temperature: float = 2.0, epochs: int = 8,
        lr: float = 5e-2, seed: int = 0, device: str = "cuda:0") -> dict[str, object]:
    """Record, train, answer. Returns the loss of every epoch and what teacher
    and student generate from the same contexts and random numbers."""
    teacher = TableTeacher(vocab, seed=seed).to(device)
    student = PairwiseTokenModel(vocab, seed=seed).to(device)
    seen = make_contexts(contexts, vocab, seed=seed).to(device)
    rec = record(teacher, seen, k, temperature=temperature)
    optimizer = FusedAdam(student.parameters(), lr=lr)
    losses = []
    for _ in range(epochs):
        total = torch.zeros((), device=device)
        for at in range(0, contexts, batch):
            rows = slice(at, at + batch)
            part = TopLogits(*(t[rows] for t in rec))
            loss = distill_step(student, optimizer, seen[rows], part, temperature=temperature)
            total += loss.detach() * len(seen[rows])
        losses.append(float(total) / contexts)
    answers = {}
    for name, model in (("teacher", teacher), ("student", student)):
        gen = torch.Generator(device=device).manual_seed(seed)
        answers[name] = generate(model, seen[:8], 12, generator=gen, top_k=50, top_p=0.9)
    return {"losses": losses, **answers}


def main() -> None:
    out = run()
    for epoch, loss in enumerate(out["losses"]):
        print(f"epoch {epoch}  loss {loss:.4f}")
    for name in ("teacher", "student"):
        tokens, log_probs = out[name]
        print(f"{name}: {tokens[0].tolist()}  mean log-probability {float(log_probs.mean()):.3f}")


if __name__ == "__main__":
    main()
