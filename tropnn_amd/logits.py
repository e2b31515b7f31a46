"""Operators on rows of logits, as hand-written HIP kernels: what a classifier
over a vocabulary needs to learn from a stronger model and to answer.

  top_logits          a teacher's record: its largest logits, their classes and
                      the log-mass of the others
  distillation_loss   the Kullback-Leibler divergence from such a record to a
                      student's logits, with its gradient
  sample_tokens       a class per row, drawn with temperature, top-k, top-p and
                      min-p from given random numbers

They have no counterpart in the reference, whose training ends in
F.cross_entropy (examples/emnist.py:221). Logits are f32, f16 or bf16
[..., vocab] on a GPU, up to 1048576 classes; leading dimensions are rows, which
may lie apart in memory (a slice of a wider tensor is read where it is). Every
sum is at least 32 bits wide. A row's order is: larger logit first, NaN before
any number, equal logits by ascending class. There is no CPU fallback: another
device raises ValueError, another type TypeError, a size past a limit
NotImplementedError.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import Tensor

from .backends.logits_hip import (
    LOGITS_DTYPES,
    MAX_TOP,
    MAX_VOCAB,
    distill_op,
    sample_hip,
    top_logits_hip,
)
from .losses import _UNITS


class TopLogits(NamedTuple):
    """A teacher's record of its k first logits per row."""

    values: Tensor  # [..., k], the logits' type, in order
    indices: Tensor  # [..., k] int64
    log_rest: Tensor  # [...] f32: log of the sum of exp(x / temperature) over the other logits


class SampledTokens(NamedTuple):
    tokens: Tensor  # [...] int64
    log_probs: Tensor  # [...] f32: under the distribution that the token was drawn from


def _check_logits(name: str, logits: Tensor) -> None:
    if logits.device.type != "cuda":
        raise ValueError(f"{name} needs logits on a GPU, got {logits.device}")
    if logits.dtype not in LOGITS_DTYPES:
        raise TypeError(f"{name} needs f32, f16 or bf16 logits, got {logits.dtype}")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{name} needs logits [..., vocab] with at least one class, got {tuple(logits.shape)}")
    if logits.shape[-1] > MAX_VOCAB:
        raise NotImplementedError(f"{name} supports up to {MAX_VOCAB} classes, got {logits.shape[-1]}")


def _check_other(name: str, what: str, t: Tensor, logits: Tensor, shape: tuple[int, ...], dtypes) -> None:
    if t.device != logits.device:
        raise ValueError(f"{name} needs {what} on {logits.device}, got {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} needs {what} of {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} needs {what} {tuple(shape)}, got {tuple(t.shape)}")


def _check_temperature(name: str, temperature: float) -> float:
    temperature = float(temperature)
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"{name} needs a positive temperature, got {temperature}")
    return temperature


def top_logits(logits: Tensor, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The k (up to 1024) first logits of every row, in order, and the log-mass
    of the others at `temperature`, the one that the record will be distilled
    at. Not differentiable: a record is a teacher's answer."""
    _check_logits("top_logits", logits)
    k = int(k)
    if not 1 <= k <= logits.shape[-1]:
        raise ValueError(f"top_logits needs 1 <= k <= {logits.shape[-1]} classes, got {k}")
    if k > MAX_TOP:
        raise NotImplementedError(f"top_logits supports k up to {MAX_TOP}, got {k}")
    return TopLogits(*top_logits_hip(logits.detach(), k, _check_temperature("top_logits", temperature)))


def distillation_loss(
    logits: Tensor,
    values: Tensor,
    indices: Tensor,
    log_rest: Tensor | None = None,
    *,
    weights: Tensor | None = None,
    temperature: float = 1.0,
    scale: float = 1.0,
    reduction: str = "mean",
) -> Tensor:
    """The divergence KL(teacher || student) at `temperature`, times its square
    (which keeps the gradient's size), from a teacher's top logits.

    logits [..., vocab]: the student's. values [..., k] (f32, f16 or bf16) and
    indices [..., k] int64: the teacher's list per row, as top_logits gives it; an
    entry of a negative index is no part of it, so rows may have shorter lists,
    and a row without any has no loss and no gradient. A row's classes are
    distinct; a class past the vocabulary makes the row's loss NaN.
    log_rest [...] f32: the log-mass of the teacher's other logits at this
    temperature. The classes outside the list then count as one class more, of
    the teacher's and of the student's remaining mass. Without it the teacher's
    distribution is the softmax of its list.
    weights [...] f32: a weight per row (0: the row is left out, whatever it holds).
    reduction: "mean", the weighted rows' sum over the sum of the weights (NaN
    where that is 0), or "sum". scale multiplies the result.

    Gradients flow to the logits alone, once: a derivative of the gradient
    (create_graph) raises RuntimeError where it is asked for, a forward-mode
    derivative NotImplementedError. Loss and gradient come from one launch
    over the rows, which also reads them only once from memory where they fit
    the caches; without a gradient asked for, the loss alone is computed. The
    backward pass from a gradient of one (loss.backward(), or a sum of losses'
    backward) leaves it at that; another value costs a pass over the gradient
    (16-bit ones are computed again, with that value before their rounding, so
    that a loss scaled against underflow keeps its small gradients), which
    `scale` spares."""
    name = "distillation_loss"
    _check_logits(name, logits)
    lead = logits.shape[:-1]
    if values.ndim < 1 or values.shape[-1] < 1:
        raise ValueError(f"{name} needs at least one list entry a row, got values {tuple(values.shape)}")
    k = values.shape[-1]
    if k > MAX_TOP:
        raise NotImplementedError(f"{name} supports lists of up to {MAX_TOP}, got {k}")
    _check_other(name, "values", values, logits, (*lead, k), tuple(LOGITS_DTYPES))
    _check_other(name, "indices", indices, logits, (*lead, k), (torch.int64,))
    if log_rest is not None:
        _check_other(name, "log_rest", log_rest, logits, lead, (torch.float32,))
        log_rest = log_rest.detach()
    if weights is not None:
        _check_other(name, "weights", weights, logits, lead, (torch.float32,))
        weights = weights.detach()
    if reduction not in ("mean", "sum"):
        raise ValueError(f"{name} needs reduction 'mean' or 'sum', got {reduction!r}")
    return distill_op()(logits, values.detach(), indices, log_rest, weights, _check_temperature(name, temperature),
                        float(scale), reduction == "mean", _UNITS.get((logits.device, torch.float32)))


def sample_tokens(
    logits: Tensor,
    uniforms: Tensor,
    *,
    temperature: float | Tensor = 1.0,
    top_k: int | Tensor = 0,
    top_p: float | Tensor = 1.0,
    min_p: float | Tensor = 0.0,
) -> SampledTokens:
    """One class per row of logits [..., vocab], from uniforms [...] f32 in [0, 1).

    temperature: divides the logits; 0 or less takes the first logit of the order
    (log-probability 0). Then, each on what the one before left: top_k keeps the
    first top_k logits of the order (0: all); top_p the shortest prefix of the
    order that holds that share of the mass (1: all); min_p the classes of at
    least min_p times the largest probability (0: all). The class is the first
    one, by index, at which the kept classes' running sum passes the row's
    uniform number times their mass. Each parameter is one value, or a tensor [...]
    with every row's own (f32; top_k int32 or int64).

    top_k up to 1024 as one value, and up to 256 as a row's own in any batch,
    draws from a short list; a larger one may search the row instead, which reads
    it several times. Not differentiable: log_probs is a number, no function of
    the logits to train through.

    Probabilities are whole multiples of 2^-40 of the row's largest, so all
    sums are exact: a row's answer depends on that row and its number alone, not
    on the batch around it or on how the work is split. A row with a NaN, or
    with all logits -inf, has token -1 and log-probability NaN."""
    name = "sample_tokens"
    _check_logits(name, logits)
    lead = logits.shape[:-1]
    _check_other(name, "uniforms", uniforms, logits, lead, (torch.float32,))
    floats = {"temperature": temperature, "top_p": top_p, "min_p": min_p}
    for what, value in floats.items():
        if isinstance(value, Tensor):
            _check_other(name, what, value, logits, lead, (torch.float32,))
            floats[what] = value.detach()
        else:
            floats[what] = value = float(value)
            if what == "temperature" and (value != value or value == math.inf):
                raise ValueError(f"{name} needs a finite temperature, got {value}")
            if what == "top_p" and not value > 0.0:
                raise ValueError(f"{name} needs top_p above 0 (1 or more: off), got {value}")
            if what == "min_p" and not 0.0 <= value <= 1.0:
                raise ValueError(f"{name} needs min_p in [0, 1], got {value}")
    if isinstance(top_k, Tensor):
        _check_other(name, "top_k", top_k, logits, lead, (torch.int32, torch.int64))
        top_k = top_k.clamp(0, MAX_VOCAB).to(torch.int32) if top_k.dtype == torch.int64 else top_k
    else:
        top_k = min(max(int(top_k), 0), MAX_VOCAB)
    return SampledTokens(*sample_hip(logits.detach(), uniforms, floats["temperature"], top_k, floats["top_p"], floats["min_p"]))
