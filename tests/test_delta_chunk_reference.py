"""The tests' two float64 forms of the gated delta rule, token by token and by chunks, are one rule."""
import pytest
import torch

import delta_chunk_reference as chunks
import delta_reference as tokens
import delta_slow_inputs as slow


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


@pytest.mark.parametrize("case", slow.CASES, ids=slow.IDS)
def test_slow_inputs_show_a_wrong_transition_of_a_segment(case):
    """With the true transition the rule by segments is the rule; with one that is 0, the identity, transposed or that of
    its diagonal alone, the state after the segments, the outputs and the first state's gradient are at least 1 % off
    (the kernels' results on these inputs are held to 5e-5 and less)."""
    q, k, v, do, beta, lg, S0, dS, m = slow.inputs(*case)
    S0 = S0.double().requires_grad_(True)

    def run(**plant):
        o, S = slow.by_segments(q, k, v, beta, lg, m, 0.125, S0, 640, **plant)
        grad = torch.autograd.grad((o * tokens.clean(do, m)).sum() + (S * dS.double()).sum(), S0)[0]
        return o.detach(), S.detach(), grad

    whole = chunks.forward(q, k, v, beta, lg, m, 0.125, S0.detach())
    grad = chunks.gradients(q, k, v, beta, lg, m, 0.125, S0.detach(), do, dS)[5]
    want = whole + (grad,)
    for a, b in zip(run(), want):
        assert float((a - b).norm()) < 1e-11 * float(b.norm())
    for plant in (torch.zeros_like, lambda M: torch.eye(M.shape[-1], dtype=M.dtype).expand_as(M), lambda M: M.mT,
                  lambda M: torch.diag_embed(torch.diagonal(M, dim1=-2, dim2=-1))):
        for a, b in zip(run(transition=plant), want):
            assert float((a - b).norm()) > 0.01 * float(b.norm())
