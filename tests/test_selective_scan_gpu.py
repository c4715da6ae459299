"""The selective scan (ops.selective_scan_forward / _backward, SelectiveScanStep) against its definition in float64.

Tolerances, relative in the 2-norm over a tensor. A result rounded once is off by at most half a step, u = eps / 2 of its type.
Inside everything is float32: dt is off by about 4 x 2^-24 (softplus of a rounded sum), a - 1 by as much again, and a step
adds four roundings; a state remembers the errors of its last 1 / (1 - a) tokens as it remembers the tokens, so that they
stay relative to it: 16 x 2^-24 = 1e-6. The adjoint goes through the same number again, sums over channels and tokens
of up to 2^14 terms add at most sqrt(2^14) x 2^-24 / 2 = 4e-6 in the mean square: 6e-6 for gradients.
"""
import pytest
import torch

import block_reference as ref
from subq_audio import ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FWD, BWD = 1e-6, 6e-6


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else 0.0


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n, d = float(b.norm()), float((a - b).norm())
    return d / n if n > 0 else d


def inputs(B, L, D, N, G, dtype, seed=0, gate=True, skip=True, bias=True, state=True, layout="plain"):
    g = torch.Generator().manual_seed(seed)
    t = T[dtype]

    def seq(*tail):
        x = torch.randn(B, L, *tail, generator=g)
        if layout == "odd":  # rows that start on no 16-byte boundary, in a wider buffer
            wide = torch.zeros(B, L, *tail[:-1], tail[-1] + 3, dtype=t)
            wide[..., 1:tail[-1] + 1] = x.to(t)
            return wide.cuda()[..., 1:tail[-1] + 1]
        if layout == "tbd":  # tokens outermost
            return x.to(t).cuda().transpose(0, 1).contiguous().transpose(0, 1)
        return x.to(t).cuda()

    s = {"u": seq(D), "dt": seq(D), "B": seq(G, N), "C": seq(G, N)}
    s["A"] = -(torch.arange(1, N + 1).float() * torch.exp(0.1 * torch.randn(D, N, generator=g))).cuda()
    s["z"] = seq(D) if gate else None
    s["D"] = (1 + 0.1 * torch.randn(D, generator=g)).cuda() if skip else None
    s["dt_bias"] = (torch.randn(D, generator=g) - 4).cuda() if bias else None
    s["state"] = (0.5 * torch.randn(B, D, N, generator=g)).cuda() if state else None
    return s, seq(D), torch.randn(B, D, N, generator=g).cuda()


def lengths_mask(B, L, seed=3):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, L + 1, (B,), generator=g)
    lens[0] = 0  # a row that has nothing
    return (torch.arange(L)[None, :] < lens[:, None]).cuda()


def call(s, **more):
    return ops.selective_scan_forward(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], **more)


def call_back(s, dout, **more):
    return ops.selective_scan_backward(s["u"], s["dt"], s["A"], s["B"], s["C"], dout, D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], **more)


def definition(s, mask=None, softplus=True, dout=None, dstate=None):
    x = {k: None if v is None else v.double().requires_grad_(dout is not None) for k, v in s.items()}
    out, h = ref.scan(x["u"], x["dt"], x["A"], x["B"], x["C"], x["D"], x["z"], x["dt_bias"], softplus, mask, x["state"])
    if dout is None:
        return out, h
    loss = (out * dout.double()).sum() + (0 if dstate is None else (h * dstate.double()).sum())
    names = [k for k, v in x.items() if v is not None]
    return dict(zip(names, torch.autograd.grad(loss, [x[k] for k in names], allow_unused=True)))


SHAPES = [  # B, L, D, N, G
    (1, 1, 1, 1, 1), (2, 9, 5, 3, 1), (1, 31, 64, 16, 1), (2, 32, 65, 16, 1), (3, 33, 130, 16, 2), (1, 100, 24, 17, 3),
    (2, 70, 48, 32, 1), (1, 65, 40, 33, 2), (2, 40, 20, 64, 2), (1, 50, 17, 100, 1), (1, 37, 8, 128, 1), (2, 257, 96, 12, 4),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype):
    B, L, D, N, G = shape
    s, dout, dstate = inputs(B, L, D, N, G, dtype)
    handover = ops.ScanHandover()
    out, h = call(s, return_state=True, handover=handover)
    want, want_h = definition(s)
    assert rel(out, want) < FWD + half(T[dtype])
    assert rel(h, want_h) < FWD
    grads = definition(s, dout=dout, dstate=dstate)
    for hand in (handover, None):
        g = call_back(s, dout, dstate=dstate, need_dstate=True, handover=hand)
        got = {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias, "state": g.dstate}
        for k, x in got.items():
            assert rel(x, grads[k]) < BWD + half(x.dtype), k


@pytest.mark.parametrize("layout", ["odd", "tbd"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layouts_and_masks(layout, dtype):
    B, L, D, N, G = 4, 77, 72, 16, 1
    s, dout, dstate = inputs(B, L, D, N, G, dtype, layout=layout)
    mask = lengths_mask(B, L)
    mask[1] = torch.rand(L, generator=torch.Generator().manual_seed(1)).cuda() < 0.5  # holes
    grads = definition(s, mask, dout=dout, dstate=dstate)
    want, want_h = definition(s, mask)
    # what is masked is not read
    for name in ("u", "dt", "z", "B", "C"):
        s[name][~mask] = float("nan")
    dout = dout.clone()
    dout[~mask] = float("inf")
    out, h = call(s, mask=mask, return_state=True)
    assert rel(out, want) < FWD + half(T[dtype]) and rel(h, want_h) < FWD
    assert bool((out[~mask] == 0).all()) and torch.equal(h[0], s["state"][0])
    g = call_back(s, dout, mask=mask, dstate=dstate, need_dstate=True)
    for k, x in {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias, "state": g.dstate}.items():
        assert rel(x, grads[k]) < BWD + half(x.dtype), k
    assert all(bool((x[~mask] == 0).all()) for x in (g.du, g.ddt, g.dz, g.dB, g.dC))


@pytest.mark.parametrize("gate,skip,bias,softplus", [(False, True, True, True), (True, False, False, True), (False, False, False, False)])
def test_without_options(gate, skip, bias, softplus):
    s, dout, _ = inputs(2, 45, 70, 16, 1, "fp32", gate=gate, skip=skip, bias=bias, state=False)
    if not softplus:
        s["dt"] = s["dt"].abs() * 0.1
    out, h = call(s, dt_softplus=softplus, return_state=True)
    want, want_h = definition(s, softplus=softplus)
    assert rel(out, want) < FWD and rel(h, want_h) < FWD
    g = call_back(s, dout, dt_softplus=softplus)
    grads = definition(s, softplus=softplus, dout=dout)
    assert (g.dz is None) == (not gate) and (g.dD is None) == (not skip) and (g.ddt_bias is None) == (not bias) and g.dstate is None
    for k, x in {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias}.items():
        if x is not None:
            assert rel(x, grads[k]) < BWD, k


@pytest.mark.parametrize("dtype,N,L", [("bf16", 16, 2500), ("fp32", 16, 2049), ("fp32", 40, 1100)])
def test_segments(dtype, N, L):
    """Few channels and many tokens: the sequence is cut (more launches than the walk alone)."""
    s, dout, dstate = inputs(1, L, 100, N, 1, dtype)
    handover = ops.ScanHandover()
    out, h = call(s, return_state=True, handover=handover)
    assert ops.last_launches() == 2
    want, want_h = definition(s)
    assert rel(out, want) < FWD + half(T[dtype]) and rel(h, want_h) < FWD
    grads = definition(s, dout=dout, dstate=dstate)
    for hand in (handover, None):
        g = call_back(s, dout, dstate=dstate, need_dstate=True, handover=hand)
        for k, x in {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias, "state": g.dstate}.items():
            assert rel(x, grads[k]) < BWD + half(x.dtype), k


def test_slow_decay_keeps_its_bits():
    """Decays of 1 - 1e-4 over 8192 tokens at a constant step: a rounded near 1 would leave 1e-4."""
    B, L, D, N = 1, 8192, 64, 16
    s, _, _ = inputs(B, L, D, N, 1, "fp32", bias=False)
    s["dt"].fill_(1.1e-4)
    s["A"].fill_(-0.93)
    out, h = call(s, dt_softplus=False, return_state=True)
    want, want_h = definition(s, softplus=False)
    assert rel(h, want_h) < FWD and rel(out, want) < FWD


def test_growing_states_behind_zeros():
    """A above 0: factors over a segment overflow, the states of the last tokens do not.

    A growing state forgets none of its roundings, so those of up to 40 steps add up: a factor 2^y is off by 1e-7 (the exponential) and by two
    halves of a step of y (the product dt A log2 e, y < 0.6, times ln 2), the step itself by two half steps (the factor applied,
    the input added). 40 (1e-7 + 2 x 0.42 x 2^-24 + 2 x 2^-24) = 1.1e-5 beside what a state that decays may be off.
    """
    grown = 40 * (1e-7 + 2 * 0.42 * 2.0 ** -24 + 2 * 2.0 ** -24)
    s, dout, _ = inputs(1, 4096, 64, 16, 1, "fp32", state=False, gate=False)
    s["A"] = s["A"].abs() * 0.05
    s["dt"].fill_(0.3)
    s["dt_bias"] = None
    s["u"][:, :4060] = 0
    s["D"] = None
    out, h = call(s, dt_softplus=False, return_state=True)
    assert ops.last_launches() == 2
    want, want_h = definition(s, softplus=False)
    assert bool(torch.isfinite(want_h).all()) and rel(out, want) < FWD + grown and rel(h, want_h) < FWD + grown
    dout[:, 40:] = 0
    g, grads = call_back(s, dout, dt_softplus=False), definition(s, softplus=False, dout=dout)
    assert rel(g.dC, grads["C"]) < BWD + grown and bool(torch.isfinite(g.du).all()) and rel(g.du, grads["u"]) < BWD + grown


def test_extreme_steps():
    """Steps that forget everything (exp underflows), that change nothing, and softplus of far arguments."""
    s, dout, _ = inputs(2, 64, 64, 16, 1, "fp32")
    s["dt"][:, ::3] = 200.0
    s["dt"][:, 1::3] = -200.0
    out, h = call(s, return_state=True)
    want, want_h = definition(s)
    assert rel(out, want) < FWD and rel(h, want_h) < FWD
    g, grads = call_back(s, dout), definition(s, dout=dout)
    for k, x in {"u": g.du, "dt": g.ddt, "B": g.dB, "C": g.dC}.items():
        assert rel(x, grads[k]) < BWD, k


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_stream_in_pieces_and_steps(dtype):
    """Pieces of 1, 8, 9 and 40 tokens from the carried state equal one pass; so do captured steps."""
    B, L, D, N = 3, 64, 96, 16
    s, _, _ = inputs(B, L, D, N, 2, dtype)
    whole, h_whole = call(s, return_state=True)
    parts, h, at = [], s["state"], 0
    for n in (1, 8, 9, 40, 6):
        o, h = ops.selective_scan_forward(s["u"][:, at:at + n], s["dt"][:, at:at + n], s["A"], s["B"][:, at:at + n], s["C"][:, at:at + n], D=s["D"],
                                          z=s["z"][:, at:at + n], dt_bias=s["dt_bias"], state=h, return_state=True)
        parts.append(o)
        at += n
    assert rel(torch.cat(parts, 1), whole) < FWD + half(T[dtype]) and rel(h, h_whole) < FWD
    bufs = {k: torch.empty_like(s[k][:, :1]) for k in ("u", "dt", "z", "B", "C")}
    state, out = s["state"].clone(), torch.empty_like(bufs["u"])
    step = ops.SelectiveScanStep(bufs["u"], bufs["dt"], s["A"], bufs["B"], bufs["C"], out, state, D=s["D"], z=bufs["z"], dt_bias=s["dt_bias"])
    step.step()
    state.copy_(s["state"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.step()
    state.copy_(s["state"])
    for t in range(L):
        for k, x in bufs.items():
            x.copy_(s[k][:, t:t + 1])
        graph.replay()
        assert rel(out, whole[:, t:t + 1]) < 1e-5 + 2 * half(T[dtype])
    assert rel(state, h_whole) < FWD


def test_state_in_place_over_segments():
    s, _, _ = inputs(1, 2048, 64, 16, 1, "fp32")
    want = call(s, return_state=True)
    out = torch.empty_like(s["u"])
    step = ops.SelectiveScanStep(s["u"], s["dt"], s["A"], s["B"], s["C"], out, s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
    step.step()
    assert torch.equal(out, want[0]) and torch.equal(s["state"], want[1])


def test_same_bits_twice_and_on_a_stream():
    s, dout, _ = inputs(2, 300, 200, 16, 1, "bf16")
    first = call_back(s, dout, need_dstate=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call_back(s, dout, need_dstate=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_two_graphs_and_two_threads():
    import threading

    s, _, _ = inputs(1, 4096, 64, 16, 1, "bf16")
    r, _, _ = inputs(1, 4096, 64, 16, 1, "bf16", seed=5)
    wants = [call(x, return_state=True) for x in (s, r)]
    graphs, outs = [], []
    for x in (s, r):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x, return_state=True))
        graphs.append(g)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, wants):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    results = [None, None]

    def work(i, x):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                results[i] = call(x, return_state=True)
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i, x)) for i, x in enumerate((s, r))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for got, want in zip(results, wants):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_tokens_and_broadcast_inputs():
    s, _, dstate = inputs(2, 5, 64, 16, 1, "fp32")
    none = {k: (v[:, :0] if k in ("u", "dt", "z", "B", "C") else v) for k, v in s.items()}
    out, h = call(none, return_state=True)
    assert out.shape == (2, 0, 64) and torch.equal(h, s["state"])
    g = call_back(none, none["u"], dstate=dstate, need_dstate=True)
    assert torch.equal(g.dstate, dstate) and float(g.dA.abs().max()) == 0 and float(g.dD.abs().max()) == 0
    # one row of u, B and C for the whole batch
    wide = dict(s, u=s["u"][:1].expand(2, -1, -1), B=s["B"][:1].expand(2, -1, -1, -1), C=s["C"][:1].expand(2, -1, -1, -1))
    out, _ = call(wide)
    assert rel(out, definition(wide)[0]) < FWD


def test_offsets_beyond_32_bits():
    """Rows further apart than 2^31 elements."""
    L, D, N = 40, 64, 16
    s, dout, _ = inputs(2, L, D, N, 1, "bf16")
    buf = torch.zeros((1 << 31) + 2 * L * D, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((2, L, D), (1 << 31, D, 1))
    far.copy_(s["u"])
    want = call(s)[0]
    got = call(dict(s, u=far))[0]
    assert torch.equal(got, want)
    a, b = call_back(s, dout), call_back(dict(s, u=far), dout)
    assert all(torch.equal(x, y) for x, y in zip(a, b) if x is not None)


def test_directional_differences():
    """The kernels' own differences along a direction: 2 eps v . grad, off by O(eps^2) and float32 rounding."""
    s, dout, _ = inputs(1, 40, 32, 16, 1, "fp32")
    g = call_back(s, dout, need_dstate=True)
    grads = {"u": g.du, "dt": g.ddt, "A": g.dA, "B": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias, "state": g.dstate}
    for k, grad in grads.items():
        v = torch.randn(s[k].shape, generator=torch.Generator().manual_seed(9)).cuda()
        eps = 1e-2
        hi = call(dict(s, **{k: s[k] + eps * v}))[0].double()
        lo = call(dict(s, **{k: s[k] - eps * v}))[0].double()
        got = float(((hi - lo) * dout.double()).sum()) / (2 * eps)
        want = float((grad.double() * v.double()).sum())
        # eps^2 / 6 of the third derivative, whose size is that of the first (exponentials and logistic functions of
        # arguments of size one), and 1e-7 / eps of the terms' sum of absolute values
        scale = float((grad.double() * v.double()).abs().sum())
        assert abs(got - want) < 2e-3 * scale + 1e-6, k


def test_refusals():
    s, dout, _ = inputs(2, 16, 64, 16, 2, "bf16")
    u = s["u"]
    with pytest.raises(RuntimeError):
        ops.selective_scan_forward(u.cpu(), s["dt"], s["A"], s["B"], s["C"])
    with pytest.raises(TypeError):
        call(dict(s, dt=s["dt"].float()))
    with pytest.raises(ValueError):
        call(dict(s, B=s["B"][..., :8]))
    with pytest.raises(ValueError):
        call(dict(s, B=s["B"].repeat(1, 1, 3, 1)[:, :, :3], C=s["C"].repeat(1, 1, 3, 1)[:, :, :3]))  # 3 groups of 64 channels
    with pytest.raises(ValueError):
        call(dict(s, A=s["A"].new_zeros(64, 129), B=u.new_zeros(2, 16, 2, 129), C=u.new_zeros(2, 16, 2, 129), state=None))
    with pytest.raises(ValueError):
        call(dict(s, state=s["state"][:1]))
    with pytest.raises(ValueError):
        call(s, mask=torch.ones(2, 15, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError):
        call(s, out=u)  # shares memory with an input
    with pytest.raises(ValueError):
        call(s, out=u.new_empty(1, 16, 64).expand(2, -1, -1))  # rows that overlap
    other = ops.ScanHandover()
    call(dict(s, u=u[:1], dt=s["dt"][:1], z=s["z"][:1], B=s["B"][:1], C=s["C"][:1], state=s["state"][:1]), handover=other)
    with pytest.raises(ValueError):
        call_back(s, dout, handover=other)
    with pytest.raises(ValueError):
        ops.SelectiveScanStep(u, s["dt"], s["A"].half(), s["B"], s["C"], torch.empty_like(u), s["state"])
    with pytest.raises(ValueError):
        ops.SelectiveScanStep(u, s["dt"], s["A"], s["B"], s["C"], torch.empty_like(u), s["state"].transpose(0, 1).contiguous().transpose(0, 1))
