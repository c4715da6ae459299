"""The selective scan at the ends of its steps' range: raw steps that are infinite, the type's lowest value, or NaN.

Tolerances as in test_selective_scan_gpu (1e-6 forward, 6e-6 gradients, half a step of a rounded result).
"""
import pytest
import torch

from test_selective_scan_gpu import BWD, FWD, T, call, call_back, definition, half, inputs, rel

pytestmark = pytest.mark.gpu

LOW = {"-inf": lambda t: float("-inf"), "lowest": lambda t: torch.finfo(t).min}


def grads_of(g):
    return {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias, "state": g.dstate}


@pytest.mark.parametrize("low", list(LOW))
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,L,D,N", [(2, 5, 70, 16), (2, 77, 70, 12), (1, 1600, 40, 16)])  # token by token, one walk, segments
def test_steps_of_nothing(B, L, D, N, dtype, low):
    """softplus of -inf (and of the type's lowest value, as a mask is written) is 0: such a token changes nothing of its channel."""
    s, dout, dstate = inputs(B, L, D, N, 1, dtype)
    off = torch.rand(B, L, D, generator=torch.Generator().manual_seed(7)).cuda() < 0.3
    off[:, 2] = True
    off[:, :, 3] = True  # a channel that never steps
    s["dt"] = torch.where(off, torch.full_like(s["dt"], LOW[low](T[dtype])), s["dt"])
    out, h = call(s, return_state=True)
    want, want_h = definition(s)
    assert bool(torch.isfinite(want).all()) and rel(out, want) < FWD + half(T[dtype]) and rel(h, want_h) < FWD
    assert torch.equal(h[:, 3], s["state"][:, 3])
    g, grads = grads_of(call_back(s, dout, dstate=dstate, need_dstate=True)), definition(s, dout=dout, dstate=dstate)
    for k, x in g.items():
        assert rel(x, grads[k]) < BWD + half(x.dtype), k
    assert float(g["dt"][off].abs().max()) == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("L", [6, 70])
def test_steps_without_end(L, dtype):
    """A raw step of +inf leaves no finite state behind, in its channel and from its token on; all else is as without it."""
    s, _, _ = inputs(2, L, 70, 16, 1, dtype)
    plain, h = call(s, return_state=True)
    dt = s["dt"].clone()
    dt[1, 4, 9] = float("inf")
    out, h_inf = call(dict(s, dt=dt), return_state=True)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[1, 4:, 9] = True
    assert torch.equal(out[~hit], plain[~hit]) and not bool(torch.isfinite(out[hit]).any())
    assert not bool(torch.isfinite(h_inf[1, 9]).any())
    h_inf[1, 9] = h[1, 9]
    assert torch.equal(h_inf, h)
    nan = s["dt"].clone()
    nan[1, 4, 9] = float("nan")
    out, _ = call(dict(s, dt=nan))
    assert torch.equal(out[~hit], plain[~hit]) and bool(torch.isnan(out[hit]).all())


def test_raw_steps_themselves():
    """dt_softplus=False: the step is the raw value, whatever softplus would make of it."""
    s, _, _ = inputs(1, 40, 33, 16, 1, "fp32", bias=False)
    s["dt"] = s["dt"].abs() * 0.1
    s["dt"][:, ::3] = 0
    out, h = call(s, dt_softplus=False, return_state=True)
    want, want_h = definition(s, softplus=False)
    assert rel(out, want) < FWD and rel(h, want_h) < FWD
