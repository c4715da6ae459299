"""The gated delta rule cut into segments whose transitions count (delta_slow_inputs.py), against float64; tolerances as in
test_delta_long_gpu.py."""
import pytest
import torch

import delta_chunk_reference as ref
import delta_slow_inputs as slow
from subq_audio import ops
from test_delta_long_gpu import NAMES, rel, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", slow.CASES, ids=slow.IDS)
def test_segments_hand_the_state_on(case):
    d, e, dtype, N, lowest, masked = case
    q, k, v, do, beta, lg, S0, dS, m = (x if x is None else x.cuda() for x in slow.inputs(*case))
    gate = lg if lowest else None
    scale = d ** -0.5
    o_ref, S_ref = ref.forward(q, k, v, beta, lg, m, scale, S0)
    lost = S_ref - ref.forward(q, k, v, beta, lg, m, scale, None)[1]
    assert float(lost.norm()) > 0.1 * float(S_ref.norm())  # what came before the first segment is still there after the last
    ho = ops.DeltaHandover()
    o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=gate, mask=m, state=S0, return_state=True, handover=ho)
    assert ops.last_launches() == 4  # gates, segments, join, walk
    assert rel(S, S_ref) < tol(S, d) and rel(o, o_ref) < tol(o, d)
    state, out = S0.clone(), torch.empty_like(o)  # the state updated in place
    ops.GatedDeltaStep(q, k, v, beta, out, state, log_gamma=gate, mask=m).step()
    assert torch.equal(state, S) and torch.equal(out, o)
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True,
                                   need_dstate=True, handover=ho)
    assert ops.last_launches() == 4 + 1  # and dk summed over its group
    for name, a, w in zip(NAMES, got, ref.gradients(q, k, v, beta, lg, m, scale, S0, do, dS)):
        assert rel(a, w) < tol(a, d), name
