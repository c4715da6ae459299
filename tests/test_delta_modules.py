"""What SubQGatedDeltaAttention refuses when it is made."""
import pytest

from subq_audio import SubQGatedDeltaAttention


def test_heads_wider_than_the_kernels_are_refused_at_once():
    with pytest.raises(ValueError, match="256"):
        SubQGatedDeltaAttention(1024)
    with pytest.raises(ValueError, match="256"):
        SubQGatedDeltaAttention(2048, 4)
    assert SubQGatedDeltaAttention(256).head_dim == 256 and SubQGatedDeltaAttention(1024, 4).head_dim == 256
