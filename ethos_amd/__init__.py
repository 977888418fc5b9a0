"""MI355X-native ETHOS expert-layer forward: product-key routing, hypernetwork expert
generation over the unique experts, reordered execution and weighted scatter-back,
as gfx950 HIP kernels behind a C-ABI (include/ethos_hip.h).

The layer classes are drop-ins for the reference's (wrmedford/ETHOS model.py and
kernels.py); see ethos_amd.layer.  Around them stand the operators of a training step: the loss over the
vocabulary, the embedding, the experts' balance and gradient clipping; see ethos_amd.training.  The model is
served from a cache of latents in pages; see ethos_amd.serving.
"""
from .layer import (  # noqa: F401
    EthosExpertLayer,
    ExpertGenerationNetwork,
    FusedLowRankMoE_Reordered,
    ProductKeyRouter,
    SimplifiedHypernetMoE,
)
from .serving import LatentCache, copy_pages, latent_append, paged_attention, verify_drafts  # noqa: F401
from .training import balance_loss, clip_grads, embedding, linear_cross_entropy  # noqa: F401

__all__ = [
    "EthosExpertLayer",
    "ExpertGenerationNetwork",
    "FusedLowRankMoE_Reordered",
    "LatentCache",
    "ProductKeyRouter",
    "SimplifiedHypernetMoE",
    "balance_loss",
    "clip_grads",
    "copy_pages",
    "embedding",
    "latent_append",
    "linear_cross_entropy",
    "paged_attention",
    "verify_drafts",
]
