"""The selective scan's backward where the parts of dB and dC pass their bound and the walk goes in ranges of tokens.

Tolerances as in test_selective_scan_gpu (6e-6 for gradients, half a step of a rounded one); two forms of the same gradient are apart by
twice that.
"""
import pytest
import torch

from subq_audio import ops
from test_selective_scan_gpu import BWD, call, call_back, definition, half, inputs, rel

pytestmark = pytest.mark.gpu


def named(g):
    return {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias, "state": g.dstate}


def definition_by_channels(s, G, mask, dout, dstate, most=2000):
    """The definition's gradients, some channels at a time; dB and dC are sums over them."""
    D = s["u"].shape[2]
    out = {k: torch.zeros(v.shape, dtype=torch.float64, device=v.device) for k, v in s.items()}
    for g in range(G):
        for a in range(g * D // G, (g + 1) * D // G, most):
            c, b = slice(a, min(a + most, (g + 1) * D // G)), slice(g, g + 1)
            part = {k: v[:, :, b] if k in ("B", "C") else v[c] if k in ("A", "D", "dt_bias") else v[:, c] if k == "state" else v[..., c] for k, v in s.items()}
            for k, x in definition(part, mask, dout=dout[..., c], dstate=dstate[:, c]).items():
                if k in ("B", "C"):
                    out[k][:, :, b] += x
                else:
                    (out[k][c] if k in ("A", "D", "dt_bias") else out[k][:, c] if k == "state" else out[k][..., c]).copy_(x)
    return out


@pytest.mark.parametrize("dtype,shape", [("fp32", (1, 601, 14100, 128, 2)), ("bf16", (3, 301, 9400, 100, 1))])
def test_ranges_against_the_definition(dtype, shape):
    B, L, D, N, G = shape
    s, dout, dstate = inputs(B, L, D, N, G, dtype)
    mask = None
    if B > 1:
        mask = torch.arange(L, device="cuda")[None, :] < torch.tensor([[L], [123], [0]], device="cuda")
    handover = ops.ScanHandover()
    call(s, mask=mask, handover=handover)
    g = call_back(s, dout, mask=mask, dstate=dstate, need_dstate=True, handover=handover)
    assert ops.last_launches() > 4  # (segments' adjoints, a walk, two sums: what one range takes)
    again = call_back(s, dout, mask=mask, dstate=dstate, need_dstate=True)
    assert all(torch.equal(a, b) for a, b in zip(g, again))
    grads = definition_by_channels(s, G, mask, dout, dstate)
    for k, x in named(g).items():
        assert rel(x, grads[k]) < BWD + half(x.dtype), k


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ranges_of_segments_against_pieces(dtype):
    """A long sequence of few channels: ranges within segments, against pieces below the bound, chained by hand."""
    B, L, D, N = 1, 140001, 64, 128
    s, dout, dstate = inputs(B, L, D, N, 1, dtype)
    seq = ("u", "dt", "z", "B", "C")
    starts = [0, 50000, 100000, L]
    states = [s["state"]]
    for a, b in zip(starts[:-2], starts[1:-1]):
        states.append(call(dict({k: (v[:, a:b] if k in seq else v) for k, v in s.items()}, state=states[-1]), return_state=True)[1])
    whole = call_back(s, dout, dstate=dstate, need_dstate=True)
    assert ops.last_launches() > 6
    parts, carry = [], dstate
    for i in (2, 1, 0):
        a, b = starts[i], starts[i + 1]
        g = call_back(dict({k: (v[:, a:b] if k in seq else v) for k, v in s.items()}, state=states[i]), dout[:, a:b], dstate=carry, need_dstate=True)
        assert ops.last_launches() <= 6
        parts.insert(0, named(g))
        carry = g.dstate
    for k, x in named(whole).items():
        if k in seq:
            want = torch.cat([p[k] for p in parts], 1)
        elif k == "state":
            want = carry
        else:
            want = sum(p[k].double() for p in parts)
        assert rel(x, want) < 2 * (BWD + half(x.dtype)), k


def test_ranges_in_a_graph():
    s, dout, dstate = inputs(1, 600, 14100, 128, 1, "bf16")
    want = call_back(s, dout, dstate=dstate, need_dstate=True)
    assert ops.last_launches() > 4
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call_back(s, dout, dstate=dstate, need_dstate=True)
    for t in held:
        t.fill_(float("nan"))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
