"""The gated delta rule where nothing is forgotten quickly, against float64 (delta_chunk_reference.py).

Tolerances, relative in the 2-norm. A tensor-core instruction cuts its sum off where an addition rounds it: up to
2^-23 of the accumulator, always towards zero, so these errors add up. A product over d has d / 16 instructions with
large terms, each product on its own fresh accumulator; between the inputs and a gradient lie ten products at most
(five in each walk: K S, Y R, K^T W, Q S, P W and their mirror images). The rest, roundings that do not add up, is
5e-7 (eight of 2^-24 in the mean square; operands are held in three bf16 planes). An output in 16 bits is rounded once
more, by eps / 2.
"""
import pytest
import torch

import delta_chunk_reference as ref
from subq_audio import ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NAMES = ("dq", "dk", "dv", "dbeta", "dlog_gamma", "dstate")


def tol(x, d):
    inside = 10 * max(4, -(-d // 16)) * 2.0 ** -23 + 5e-7
    return inside + (torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0)


def rel(a, b):
    assert a.shape == b.shape
    return float((a.double() - b.double()).norm() / b.double().norm())


def inputs(B, H, Hk, N, d, e, dtype, seed, low, high):
    """Unit keys, beta between low and high, a state of ordinary size."""
    g = torch.Generator().manual_seed(seed)

    def heads(h, w, unit):
        x = torch.randn(B, N, h, w, generator=g)
        return (x / x.norm(dim=-1, keepdim=True) if unit else x).to(T[dtype]).cuda().transpose(1, 2)

    q, k, v, do = heads(H, d, True), heads(Hk, d, True), heads(H, e, False), heads(H, e, False)
    beta = (low + (high - low) * torch.rand(B, H, N, generator=g)).cuda()
    return q, k, v, do, beta, torch.randn(B, H, d, e, generator=g).cuda(), torch.randn(B, H, d, e, generator=g).cuda()


@pytest.mark.parametrize("B,H,N,d,e,dtype", [(1, 2, 16384, 64, 64, "fp32"), (1, 2, 16384, 64, 64, "bf16"), (1, 40, 16384, 64, 64, "bf16"),
                                             (1, 2, 16384, 64, 32, "fp16"), (1, 76, 8192, 128, 32, "fp32"), (1, 1, 16384, 100, 64, "bf16")])
def test_a_state_that_lasts_keeps_its_bits(B, H, N, d, e, dtype):
    """No decay and small beta: the state after 16384 tokens still holds most of the one before them. What a chunk adds
    must not cost the state a rounding in one direction at every instruction (1e-4 in all)."""
    q, k, v, do, beta, S0, dS = inputs(B, H, 1, N, d, e, dtype, N + d + H, 0.001, 0.004)
    lg = torch.zeros_like(beta)
    o_ref, S_ref = ref.forward(q, k, v, beta, lg, None, d ** -0.5, S0)
    from_zero = ref.forward(q, k, v, beta, lg, None, d ** -0.5, None)[1]
    assert float((S_ref - from_zero).norm()) > 0.2 * float(S_ref.norm())  # the state before the first token is still there
    ho = ops.DeltaHandover()
    o, S = ops.gated_delta_forward(q, k, v, beta, state=S0, return_state=True, handover=ho)
    assert rel(S, S_ref) < tol(S, d) and rel(o, o_ref) < tol(o, d)
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True, handover=ho)
    for name, a, w in zip(NAMES, got, ref.gradients(q, k, v, beta, lg, None, d ** -0.5, S0, do, dS)):
        assert rel(a, w) < tol(a, d), name


@pytest.mark.parametrize("lowest", [-9.02e-5, -6.6e-5, -3.88e-5])
@pytest.mark.parametrize("B,H,N,d,e,dtype", [(1, 2, 16384, 64, 64, "fp32"), (1, 76, 16384, 64, 32, "bf16")])
def test_a_slow_decay_keeps_its_bits(B, H, N, d, e, dtype, lowest):
    """The same decay at every token: what a chunk leaves of the state is near 1, and a rounding of it must not be the same
    one 256 times over (2^-25 at the worst, as at these)."""
    q, k, v, do, beta, S0, dS = inputs(B, H, 1, N, d, e, dtype, N + d, 0.0005, 0.001)
    lg = torch.full_like(beta, lowest)
    _, S_ref = ref.forward(q, k, v, beta, lg, None, d ** -0.5, S0)
    _, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, state=S0, return_state=True)
    assert rel(S, S_ref) < 3e-6  # 256 roundings that do not add up, 16 x 2^-24, and 2e-6 as in test_delta_gpu.py
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, state=S0, dstate=dS, need_dstate=True)
    want = ref.gradients(q, k, v, beta, lg, None, d ** -0.5, S0, do, dS)
    assert rel(got[5], want[5]) < 3e-6
