"""Neural-network module aliases (reference python/subq_audio/nn.py)."""
from .autograd import SubQAttentionFunction, SubQLinearAttention
from .delta import SubQGatedDeltaAttention, SubQLayerNorm
from .state_space import SubQFp8Linear, SubQRMSNorm, SubQSelectiveStateSpace, SubQStateSpaceBlock

SubQuadraticAttention = SubQLinearAttention

__all__ = ["SubQLinearAttention", "SubQuadraticAttention", "SubQAttentionFunction", "SubQGatedDeltaAttention",
           "SubQLayerNorm", "SubQSelectiveStateSpace", "SubQStateSpaceBlock", "SubQRMSNorm", "SubQFp8Linear"]
