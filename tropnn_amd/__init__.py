"""MI355X-native PairwiseLinear: `PairwiseLinear(..., backend="hip")` runs the
comparator route, LUT gather-sum and min-margin STE backward as gfx950 HIP
kernels in libtropnn_hip.so (C ABI: include/tropnn_hip.h)."""
from .backends import has_pairwise_hip, pairwise_hip, pairwise_hip_forward, pairwise_hip_route
from .layers import PairwiseLinear, RoutedLinearBase
from .logits import SampledTokens, TopLogits, distillation_loss, sample_tokens, top_logits
from .losses import cross_entropy, unit_gradient
from .optim import FusedAdam, FusedAdamW

__all__ = [
    "FusedAdam",
    "FusedAdamW",
    "PairwiseLinear",
    "RoutedLinearBase",
    "SampledTokens",
    "TopLogits",
    "cross_entropy",
    "distillation_loss",
    "has_pairwise_hip",
    "pairwise_hip",
    "pairwise_hip_forward",
    "pairwise_hip_route",
    "sample_tokens",
    "top_logits",
    "unit_gradient",
]
