"""SubQLayerNorm and SubQGatedDeltaAttention at the edges of what they stand in for."""
import pytest
import torch

from subq_audio import SubQLayerNorm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_refuses_another_width_as_torch_does(affine):
    for norm in (torch.nn.LayerNorm(64, elementwise_affine=affine).cuda(), SubQLayerNorm(64, elementwise_affine=affine).cuda()):
        for shape in ((3, 32), (3, 128), (64, 3), (2, 1)):
            with pytest.raises((RuntimeError, ValueError)):
                norm(torch.randn(*shape, device="cuda"))
        assert norm(torch.randn(5, 64, device="cuda")).shape == (5, 64)
