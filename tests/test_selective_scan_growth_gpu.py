"""States of the selective scan that grow (A above 0) past 2^127 times within a few tokens, over zeros: what is 0 stays 0.

Tolerances as in test_selective_scan_gpu beside what a growing state keeps of its roundings, derived below.
"""
import pytest
import torch

from subq_audio import ops
from test_selective_scan_gpu import BWD, FWD, call, call_back, definition, inputs, rel

pytestmark = pytest.mark.gpu


def growing(L, D):
    """A dt between 0.2 and 6.5: 32 tokens grow a state up to e^200 times."""
    s, dout, _ = inputs(1, L, D, 16, 1, "fp32", gate=False, skip=False, bias=False, state=False)
    s["A"] = (s["A"].abs() / s["A"].abs().max() * 21).clamp_min(0.7)
    s["dt"].fill_(0.3)
    s["u"].zero_()
    return s, dout


# A factor 2^y, y = dt A log2 e below 9.1, is off by 1e-7 (the exponential) and by two halves of a step of y times ln 2, the step itself by two
# half steps; 12 such steps stand between the first input and the last. A segment's sum has y of the whole stretch, 110 at most, in
# one exponential: two halves of a step of it (the sum of steps and the product), times ln 2.
GROWN = 12 * (1e-7 + 2 * 9.1 * 0.7 * 2.0 ** -24 + 2 * 2.0 ** -24) + 2 * 110 * 0.7 * 2.0 ** -24


@pytest.mark.parametrize("at", [4084, 2050, 100])
def test_states_that_grow_within_a_tile(at):
    """Inputs in 12 tokens only, and no step behind them; over the zeros before them the factors pass 2^127 within a tile."""
    s, _ = growing(4096, 64)
    s["u"][:, at:at + 12] = torch.randn(1, 12, 64, generator=torch.Generator().manual_seed(2)).cuda()
    s["dt"][:, at + 12:] = 0
    out, h = call(s, dt_softplus=False, return_state=True)
    assert ops.last_launches() == 2
    want, want_h = definition(s, softplus=False)
    assert bool(torch.isfinite(want_h).all())
    assert rel(out, want) < FWD + GROWN and rel(h, want_h) < FWD + GROWN


@pytest.mark.parametrize("at", [0, 2050, 3900])
def test_adjoints_that_grow_within_a_tile(at):
    """The same backwards: no step before 12 tokens whose outputs alone count."""
    s, dout = growing(4096, 64)
    s["state"] = torch.zeros(1, 64, 16, device="cuda")
    s["dt"][:, :at] = 0
    dout[:, :at] = 0
    dout[:, at + 12:] = 0
    g = call_back(s, dout, dt_softplus=False, need_dstate=True)
    grads = definition(s, softplus=False, dout=dout)
    assert bool(torch.isfinite(grads["state"]).all()) and bool(torch.isfinite(grads["u"]).all())
    assert rel(g.du, grads["u"]) < BWD + GROWN and rel(g.dstate, grads["state"]) < BWD + GROWN
