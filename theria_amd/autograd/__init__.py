"""autograd.Functions: the HIP operators (SDPAOp / SDPABackwardOp, layer norm, embedding, linear cross entropy) and the
pure-PyTorch references."""

from .graphed_hvp import GraphedSDPAHVP
from .hip_embedding import hip_embedding
from .hip_layer_norm import hip_layer_norm
from .hip_linear_ce import hip_linear_cross_entropy
from .hip_sdpa import SDPABackwardOp, SDPAOp, hip_sdpa, hip_sdpa_hvp, hip_sdpa_with_lse
from .sdpa_custom_function import SDPACustom
from .sdpa_function import SDPAFunction, sdpa

__all__ = ["SDPAOp", "SDPABackwardOp", "hip_sdpa", "hip_sdpa_with_lse", "hip_sdpa_hvp", "GraphedSDPAHVP", "SDPACustom", "SDPAFunction", "sdpa",
           "hip_layer_norm", "hip_embedding", "hip_linear_cross_entropy"]
