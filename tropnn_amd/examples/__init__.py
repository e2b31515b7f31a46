"""Callers of the PairwiseLinear path: the pairwise family of the reference's
EMNIST classifier (examples/emnist.py). tropnn_amd.examples.distill, a token
model that learns from a teacher's top logits and answers by sampling, runs by
itself (python -m tropnn_amd.examples.distill)."""
from .emnist import EmnistPairwiseClassifier, make_c5_batch, train_step

__all__ = ["EmnistPairwiseClassifier", "make_c5_batch", "train_step"]
