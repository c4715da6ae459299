"""The short causal convolution (ops.causal_conv_forward / _backward, CausalConvStep) against its definition in float64.

Tolerances, relative in the 2-norm: half a step of the result's type, u = eps / 2; inside at most 4 products, a bias and a
logistic function in float32, 10 x 2^-24 = 6e-7 (1e-6); the backward twice that, and its sums over up to 2^12 tokens, 64
of them in a row before they are added with their rounding kept, 8 x 2^-24 in the mean square: 3e-6.
"""
import pytest
import torch

import block_reference as ref
from subq_audio import ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FWD, BWD = 1e-6, 3e-6


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else 0.0


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n, d = float(b.norm()), float((a - b).norm())
    return d / n if n > 0 else d


def inputs(B, L, D, W, dtype, seed=0, bias=True, state=True, layout="plain"):
    g = torch.Generator().manual_seed(seed)
    t = T[dtype]

    def seq():
        x = torch.randn(B, L, D, generator=g).to(t)
        if layout == "half":  # one half of a projection's output
            return torch.cat([x, x], -1).cuda()[..., :D]
        if layout == "odd":
            wide = torch.zeros(B, L, D + 3, dtype=t)
            wide[..., 1:D + 1] = x
            return wide.cuda()[..., 1:D + 1]
        return x.cuda()

    x, dout = seq(), seq()
    w = (torch.randn(D, W, generator=g) / W ** 0.5).cuda()
    b = (0.3 * torch.randn(D, generator=g)).cuda() if bias else None
    S, dS = (torch.randn(B, W - 1, D, generator=g).to(t).cuda() for _ in range(2))
    return x, w, b, S if state else None, dout, dS


def definition(x, w, b, S, act, mask, dout=None, dS=None):
    leaves = [None if v is None else v.double().requires_grad_(True) for v in (x, w, b, S)]
    y, win = ref.conv(leaves[0], leaves[1], leaves[2], act, mask, leaves[3])
    if dout is None:
        return y.detach(), win.detach()
    loss = (y * dout.double()).sum() + (0 if dS is None else (win * dS.double()).sum())
    live = [v for v in leaves if v is not None]
    got = iter(torch.autograd.grad(loss, live, allow_unused=True))
    return [None if v is None else next(got) for v in leaves]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,L,D,W,layout", [(1, 1, 1, 2, "plain"), (2, 2, 8, 4, "plain"), (1, 8, 40, 3, "plain"), (2, 9, 64, 4, "half"), (3, 31, 33, 4, "plain"),
                                            (2, 32, 48, 2, "odd"), (2, 65, 136, 3, "half"), (1, 130, 264, 4, "plain"), (2, 100, 17, 4, "odd")])
def test_forward_and_backward(B, L, D, W, layout, dtype):
    for act, bias, state in (("silu", True, True), (None, False, False)):
        x, w, b, S, dout, dS = inputs(B, L, D, W, dtype, bias=bias, state=state, layout=layout)
        y, win = ops.causal_conv_forward(x, w, b, activation=act, state=S, return_state=True)
        want, want_win = definition(x, w, b, S, act, None)
        assert rel(y, want) < FWD + half(T[dtype])
        assert torch.equal(win.double(), want_win)
        got = ops.causal_conv_backward(x, w, dout, b, activation=act, state=S, dstate=dS, need_dstate=state)
        for name, a, e in zip(("dx", "dw", "db", "dstate"), got, definition(x, w, b, S, act, None, dout, dS)):
            if e is None:
                assert a is None or (name == "dstate" and not state), name
            else:
                assert rel(a, e) < BWD + half(a.dtype), name


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("L", [7, 8, 9, 40, 200])
def test_masks(L, dtype):
    B, D, W = 5, 40, 4
    x, w, b, S, dout, dS = inputs(B, L, D, W, dtype)
    mask = torch.zeros(B, L, dtype=torch.bool)
    mask[1, :L // 2] = True   # padded behind
    mask[2, L - 2:] = True    # padded in front
    mask[3, :1] = True        # one token
    mask[4] = torch.rand(L, generator=torch.Generator().manual_seed(2)) < 0.6  # holes
    mask = mask.cuda()
    want, want_win = definition(x, w, b, S, "silu", mask)
    grads = definition(x, w, b, S, "silu", mask, dout, dS)
    x, dout = x.clone(), dout.clone()
    x[~mask] = float("nan")
    dout[~mask] = float("-inf")
    y, win = ops.causal_conv_forward(x, w, b, mask=mask, state=S, return_state=True)
    assert rel(y, want) < FWD + half(T[dtype]) and bool((y[~mask] == 0).all())
    assert torch.equal(win.double(), want_win) and torch.equal(win[0], S[0])
    got = ops.causal_conv_backward(x, w, dout, b, mask=mask, state=S, dstate=dS, need_dstate=True)
    for name, a, e in zip(("dx", "dw", "db", "dstate"), got, grads):
        assert rel(a, e) < BWD + half(a.dtype), name
    assert bool((got[0][~mask] == 0).all())


def test_stream_in_pieces_and_captured_steps():
    B, L, D, W = 3, 60, 96, 4
    x, w, b, S, _, _ = inputs(B, L, D, W, "bf16", layout="half")
    whole, win_whole = ops.causal_conv_forward(x, w, b, state=S, return_state=True)
    win, at, parts = S, 0, []
    for n in (1, 2, 3, 8, 9, 37):
        y, win = ops.causal_conv_forward(x[:, at:at + n], w, b, state=win, return_state=True)
        parts.append(y)
        at += n
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(win, win_whole)
    buf, out, state = torch.empty(B, 1, D, dtype=x.dtype, device="cuda"), torch.empty(B, 1, D, dtype=x.dtype, device="cuda"), S.clone()
    step = ops.CausalConvStep(buf, w, b, out, state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.step()
    state.copy_(S)
    for t in range(L):
        buf.copy_(x[:, t:t + 1])
        graph.replay()
        assert torch.equal(out, whole[:, t:t + 1])
    assert torch.equal(state, win_whole)


def test_long_in_place_and_none():
    """A window updated in place by a call of many tokens; no tokens at all; the same bits twice."""
    x, w, b, S, dout, dS = inputs(2, 500, 64, 4, "fp32")
    y, win = ops.causal_conv_forward(x, w, b, state=S, return_state=True)
    out, state = torch.empty_like(x), S.clone()
    ops.CausalConvStep(x, w, b, out, state).step()
    assert torch.equal(out, y) and torch.equal(state, win)
    y, win = ops.causal_conv_forward(x[:, :0], w, b, state=S, return_state=True)
    assert y.shape == (2, 0, 64) and torch.equal(win, S)
    dx, dw, db, ds = ops.causal_conv_backward(x[:, :0], w, dout[:, :0], b, state=S, dstate=dS, need_dstate=True)
    assert torch.equal(ds, dS) and float(dw.abs().max()) == 0 and float(db.abs().max()) == 0
    first, second = (ops.causal_conv_backward(x, w, dout, b, state=S, dstate=dS, need_dstate=True) for _ in range(2))
    assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_offsets_beyond_32_bits():
    x, w, b, S, dout, _ = inputs(2, 40, 64, 4, "bf16")
    buf = torch.zeros((1 << 31) + 40 * 64, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((2, 40, 64), (1 << 31, 64, 1))
    far.copy_(x)
    assert torch.equal(ops.causal_conv_forward(far, w, b)[0], ops.causal_conv_forward(x, w, b)[0])
    assert all(torch.equal(a, c) for a, c in zip(ops.causal_conv_backward(far, w, dout, b)[:3], ops.causal_conv_backward(x, w, dout, b)[:3]))


def test_refusals():
    x, w, b, S, dout, _ = inputs(2, 16, 32, 4, "bf16")
    with pytest.raises(RuntimeError):
        ops.causal_conv_forward(x.cpu(), w)
    for bad in (torch.zeros(32, 1), torch.zeros(32, 5), torch.zeros(31, 4)):
        with pytest.raises(ValueError):
            ops.causal_conv_forward(x, bad.cuda())
    with pytest.raises(ValueError):
        ops.causal_conv_forward(x, w, activation="gelu")
    with pytest.raises(ValueError):
        ops.causal_conv_forward(x, w, state=S[:, :2])
    with pytest.raises(ValueError):
        ops.causal_conv_forward(x, w, out=x)
    with pytest.raises(TypeError):
        ops.causal_conv_forward(x.double(), w)
    with pytest.raises(TypeError):
        ops.causal_conv_backward(x, w, dout.float())
    with pytest.raises(ValueError):
        ops.CausalConvStep(x, w.half(), b, torch.empty_like(x), S)
    with pytest.raises(ValueError):
        ops.CausalConvStep(x, w, b, torch.empty_like(x), S.float())
