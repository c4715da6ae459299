"""The tests' two float64 forms of the gated delta rule, token by token and by chunks, are one rule."""
import pytest
import torch

import delta_chunk_reference as chunks
import delta_reference as tokens


@pytest.mark.parametrize("N,mask,lowest", [(1, False, -0.3), (127, True, -0.3), (300, True, -3.0), (257, False, -1e-4)])
def test_chunks_equal_tokens(N, mask, lowest):
    g = torch.Generator().manual_seed(N)
    B, H, d, e = 2, 4, 12, 7

    def randn(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64)

    q, k, v, do = randn(B, 2, N, d), randn(B, 1, N, d), randn(B, 4, N, e), randn(B, H, N, e)
    k = k / k.norm(dim=-1, keepdim=True)
    beta, lg = torch.rand(B, H, N, generator=g, dtype=torch.float64), lowest * torch.rand(B, H, N, generator=g, dtype=torch.float64)
    S0, dS = randn(B, H, d, e), randn(B, H, d, e)
    m = torch.rand(B, N, generator=g) < 0.7 if mask else None
    if mask:
        m[:, 20:60] = False
    args = (q, k, v, beta, lg, m, 0.3, S0)
    # float64: 300 steps of products of up to 12 terms stay within 1e-12 of the values
    for a, b in zip(chunks.forward(*args), tokens.forward(*args)):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)
    for a, b in zip(chunks.gradients(*args, do, dS), tokens.gradients(*args, do, dS)):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)
