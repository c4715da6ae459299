"""The gated delta rule's float32 results with 16-bit inputs are as exact as with float32 ones: operands in between are held
in three bf16 planes whatever the inputs' type. The tolerance is test_delta_gpu.py's for float32 inputs, 2e-6 in the 2-norm
(planes to 2^-24, float32 sums of up to 64 products, a factor of 4 for how the recurrence passes errors on)."""
import pytest
import torch

import delta_chunk_reference as ref
from subq_audio import ops
from test_delta_gpu import inputs, poison, rel

pytestmark = pytest.mark.gpu

CASES = [(2, 4, 4, 2, 2, 700, 64, 64, "bf16", "bnhd", "tail"), (8, 12, 12, 12, 12, 400, 64, 64, "bf16", "bnhd", None),
         (1, 2, 2, 2, 2, 4096, 64, 64, "bf16", "bhnd", "random"), (2, 4, 4, 1, 4, 500, 128, 128, "bf16", "bnhd", "tail"),
         (2, 3, 3, 3, 3, 300, 80, 48, "bf16", "odd", "random"), (1, 2, 1, 2, 2, 333, 32, 32, "bf16", "bnhd", None),
         (2, 4, 2, 4, 2, 300, 64, 128, "fp16", "bnhd", "tail"), (1, 4, 4, 4, 4, 4096, 64, 64, "fp16", "bnhd", None),
         (2, 2, 2, 2, 2, 250, 128, 64, "fp16", "bnhd", "random"), (1, 3, 3, 3, 3, 178, 32, 32, "fp16", "bnhd", None)]


@pytest.mark.parametrize("case", CASES, ids=["-".join(str(x) for x in c) for c in CASES])
def test_float32_results_of_16_bit_inputs(case):
    B, H, Hq, Hk, Hv, N, d, e, dtype, layout, mask = case
    q, k, v, do, beta, lg, S0, dS, m = inputs(B, H, Hq, Hk, Hv, N, d, e, dtype, seed=N + e, layout=layout, mask=mask)
    scale = d ** -0.5
    o_ref, S_ref = ref.forward(q, k, v, beta, lg, m, scale, S0)
    want = ref.gradients(q, k, v, beta, lg, m, scale, S0, do, dS)
    q, k, v, do, beta, lg = (poison(x, m) for x in (q, k, v, do, beta, lg))
    _, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, return_state=True, path="chunked")
    assert rel(S, S_ref) < 2e-6
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True)
    for name, a, w in list(zip(("dq", "dk", "dv", "dbeta", "dlog_gamma", "dstate"), got, want))[3:]:
        assert rel(a, w) < 2e-6, name


@pytest.mark.parametrize("dtype,d,e,N", [("fp16", 64, 1, 30), ("bf16", 64, 64, 700), ("fp32", 64, 64, 200), ("fp32", 128, 33, 64)])
def test_log_gamma_gradient_where_the_last_token_forgets_all(dtype, d, e, N):
    """What the last token writes is all that the final state has, and a large gradient of that state has nothing to do with
    any log gamma. The other terms of a token's gradient are at most 64 of the gradients' own size: 2e-6 as above."""
    q, k, v, do, beta, lg, S0, dS, _ = inputs(1, 3, 3, 1, 3, N, d, e, dtype, seed=N + e)
    lg[:, :, -1] = -30.0
    want = ref.gradients(q, k, v, beta, lg, None, 1.0, S0, 0.1 * do, 10 * dS)
    got = ops.gated_delta_backward(q, k, v, beta, 0.1 * do, log_gamma=lg, scale=1.0, state=S0, dstate=10 * dS, need_dlog_gamma=True)
    assert rel(got[4], want[4]) < 2e-6


@pytest.mark.parametrize("d,e,N,lowest", [(64, 64, 4096, -1e-4), (256, 64, 4096, -1e-3), (33, 40, 3000, -1e-3)])
def test_token_steps_with_slow_decay(d, e, N, lowest):
    """The token-recurrent kernel over thousands of tokens that hardly decay, with little written: gamma is near 1, and a
    rounding of it to float32 (2^-25) would be the same at every token, N 2^-25 in all (1.2e-4). Each token's own
    roundings of the state (2^-24 of it, two) do not add up: sqrt(N) 2^-24 in the mean square, 4e-6 for 4096 tokens, with
    a margin of 2 for what beta passes on."""
    q, k, v, do, beta, _, S0, dS, _ = inputs(1, 2, 2, 2, 2, N, d, e, "fp32", seed=d)
    lg, beta = torch.full_like(beta, lowest), 0.01 * beta
    lg[:, 1] *= 0.7
    _, S_ref = ref.forward(q, k, v, beta, lg, None, 1.0, S0)
    _, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, scale=1.0, state=S0, return_state=True, path="exact")
    assert rel(S, S_ref) < 2 * N ** 0.5 * 2.0 ** -24


@pytest.mark.parametrize("d", [64, 100, 200])
@pytest.mark.parametrize("lowest", [1.0, -0.05, -0.07, -0.6, -6.0])
def test_a_state_that_nothing_is_written_to(d, lowest):
    """beta 0: the state is the product of the decays, each within 2^-23 of itself (an exponential and a product), however
    little is left of it."""
    N = 12
    q, k, v, _, beta, _, S0, _, _ = inputs(1, 2, 2, 2, 2, N, d, 40, "fp32", seed=d)
    lg = torch.full_like(beta, lowest)
    want = S0.double() * torch.exp(lg.double().sum(-1))[..., None, None]
    for path in ("exact", "chunked") if d <= 128 else ("exact",):
        _, S = ops.gated_delta_forward(q, k, v, 0.0, log_gamma=lg, state=S0, return_state=True, path=path)
        assert float(((S.double() - want) / want).abs().max()) < 2 * N * 2.0 ** -23, path
