"""Neural-network module aliases (reference python/subq_audio/nn.py)."""
from .autograd import SubQAttentionFunction, SubQLinearAttention
from .delta import SubQGatedDeltaAttention, SubQLayerNorm

SubQuadraticAttention = SubQLinearAttention

__all__ = ["SubQLinearAttention", "SubQuadraticAttention", "SubQAttentionFunction", "SubQGatedDeltaAttention",
           "SubQLayerNorm"]
