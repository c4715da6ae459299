"""Masks in the short forms: calls of up to eight tokens and the step handles, which read the caller's mask at every step.

Tolerances as in test_selective_scan_gpu (1e-6 beside half a step of the type); the convolution's four products and the silu of
their sum are off by less.
"""
import pytest
import torch

import block_reference as ref
from subq_audio import ops
from test_selective_scan_gpu import FWD, T, call, definition, half, inputs, rel

pytestmark = pytest.mark.gpu


def holes(B, L, seed=5):
    mask = torch.rand(B, L, generator=torch.Generator().manual_seed(seed)).cuda() < 0.6
    mask[0] = False
    return mask


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("L,N", [(1, 16), (5, 16), (8, 13), (8, 40)])
def test_short_masked_scans(L, N, dtype):
    s, _, _ = inputs(4, L, 70, N, 2, dtype)
    mask = holes(4, L)
    want, want_h = definition(s, mask)
    for name in ("u", "dt", "z", "B", "C"):
        s[name][~mask] = float("nan")
    out, h = call(s, mask=mask, return_state=True)
    assert rel(out, want) < FWD + half(T[dtype]) and rel(h, want_h) < FWD
    assert bool((out[~mask] == 0).all()) and torch.equal(h[0], s["state"][0])


def streams(B, L, D, N, dtype):
    s, _, _ = inputs(B, L, D, N, 1, dtype)
    x = inputs(B, L, D, N, 1, dtype, seed=8)[0]["u"]
    w = (torch.randn(D, 4, generator=torch.Generator().manual_seed(1)) / 2).cuda()
    return s, x, w, torch.randn(B, 3, D, generator=torch.Generator().manual_seed(2)).to(T[dtype]).cuda()


@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("layout", ["rows", "time-major", "one"])
def test_steps_see_their_mask_change(layout, graph, kind):
    """One token a step, streams that pause and end: the mask's buffer is refilled between steps, whatever its strides are."""
    B, L, D, N = 3, 12, 70, 16
    s, x, w, window = streams(B, L, D, N, "fp32")
    masks = holes(B, L).to(kind)
    if layout == "one":  # the same for all streams
        masks = masks[1:2].expand(B, L)
    want, want_h = definition(s, masks.bool())
    want_y, want_w = [], window.double()  # (a window skips a stream's paused tokens: step by step)
    for t in range(L):
        y, want_w = ref.conv(x[:, t:t + 1].double(), w.double(), None, "silu", masks[:, t:t + 1].bool(), want_w)
        want_y.append(y)
    if layout == "one":
        cell = torch.ones(1, 1, dtype=kind, device="cuda")
        mask = cell.expand(B, 1)
    else:
        cell = torch.ones(4, B, dtype=kind, device="cuda")[1:2] if layout == "time-major" else torch.ones(B, 1, dtype=kind, device="cuda")
        mask = cell.t() if layout == "time-major" else cell
    bufs = {k: torch.empty_like(s[k][:, :1]) for k in ("u", "dt", "z", "B", "C")}
    xb, y, out, h = torch.empty_like(x[:, :1]), torch.empty_like(x[:, :1]), torch.empty_like(x[:, :1]), s["state"].clone()
    conv = ops.CausalConvStep(xb, w, None, y, window, mask=mask)
    scan = ops.SelectiveScanStep(bufs["u"], bufs["dt"], s["A"], bufs["B"], bufs["C"], out, h, D=s["D"], z=bufs["z"], dt_bias=s["dt_bias"], mask=mask)
    first_h, first_w = h.clone(), window.clone()
    run = lambda: (conv.step(), scan.step())  # noqa: E731
    if graph:
        run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        run = g.replay
        h.copy_(first_h)
        window.copy_(first_w)
    for t in range(L):
        for k, b in bufs.items():
            b.copy_(s[k][:, t:t + 1])
        xb.copy_(x[:, t:t + 1])
        cell.copy_(masks[:1, t:t + 1] if layout == "one" else masks[:, t:t + 1].t() if layout == "time-major" else masks[:, t:t + 1])
        run()
        assert rel(out, want[:, t:t + 1]) < 1e-5 and rel(y, want_y[t]) < 1e-5, t
    assert rel(h, want_h) < FWD and torch.equal(window.double(), want_w)


def test_time_major_masks_of_several_tokens_are_refused():
    s, x, w, window = streams(3, 4, 32, 16, "fp32")
    mask = torch.ones(4, 3, dtype=torch.bool, device="cuda").t()
    out = torch.empty_like(x)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.CausalConvStep(x, w, None, out, window, mask=mask)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.SelectiveScanStep(s["u"], s["dt"], s["A"], s["B"], s["C"], out, s["state"], mask=mask)
