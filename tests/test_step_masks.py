"""Masks of the step handles on the host (no GPU): read where they are, or refused."""
import pytest
import torch

from subq_audio import block_ops


@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
def test_a_single_tokens_mask_is_read_where_it_is(kind):
    """[B, 1] masks of any strides are passed on, not copied."""
    wide = torch.ones(5, 4, dtype=kind)
    for mask in (wide.t()[:, 1:2], wide[:4, 2:3], wide[1:2].t(), wide[:1, :1].expand(4, 1)):
        block_ops._step_mask(mask)
        at, stride = block_ops._mask(mask, 4, 1, mask.device, [])
        assert at == mask.data_ptr() and stride == mask.stride(0)
    with pytest.raises(ValueError, match="contiguous rows"):
        block_ops._step_mask(wide.t())
