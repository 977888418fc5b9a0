"""MI355X-native ETHOS expert-layer forward: product-key routing, hypernetwork expert
generation over the unique experts, reordered execution and weighted scatter-back,
as gfx950 HIP kernels behind a C-ABI (include/ethos_hip.h).

The layer classes are drop-ins for the reference's (wrmedford/ETHOS model.py and
kernels.py); see ethos_amd.layer.  Around them stand the operators of a training step: the loss over the
vocabulary, the embedding, the experts' balance and gradient clipping; see ethos_amd.training.
"""
from .layer import (  # noqa: F401
    EthosExpertLayer,
    ExpertGenerationNetwork,
    FusedLowRankMoE_Reordered,
    ProductKeyRouter,
    SimplifiedHypernetMoE,
)
from .training import balance_loss, clip_grads, embedding, linear_cross_entropy  # noqa: F401

__all__ = [
    "EthosExpertLayer",
    "ExpertGenerationNetwork",
    "FusedLowRankMoE_Reordered",
    "ProductKeyRouter",
    "SimplifiedHypernetMoE",
    "balance_loss",
    "clip_grads",
    "embedding",
    "linear_cross_entropy",
]
