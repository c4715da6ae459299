"""The selective state space layer in use: differentiable calls and modules against the definitions in float64, generation through
the state cache, the quantised block, the torch operators.

Tolerances, relative in the 2-norm. float32: the kernels' own (1e-6 forward, 6e-6 gradients) through a layer of four of them and
torch's float32 products of up to 128 terms: 2e-5. bf16: each tensor between two operators is rounded, u = 2^-9 in the mean
square (2^-8 at most); about eight of them lie between the input and the output: sqrt(8) x 2^-9 = 6e-3, and 3e-2 with what the
recurrence and the products make of them. 8 bits: every 128 of a row keep 4 significant bits, 2^-4 at most and 2.6e-2 in the mean
square, of the input and of the weights of two projections: sqrt(4) x 2.6e-2 = 5e-2, and a factor of 2: 0.1.
"""
import pytest
import torch

import block_reference as ref
from subq_audio import (SubQFp8Linear, SubQRMSNorm, SubQSelectiveStateSpace, SubQStateSpaceBlock, causal_conv, ops, rms_norm, selective_scan)
from subq_audio.cache import StateCache, run_layers

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n, d = float(b.norm()), float((a - b).norm())
    return d / n if n > 0 else d


def layer(hidden=48, seed=0, **k):
    torch.manual_seed(seed)
    return SubQSelectiveStateSpace(hidden, **k).cuda()


def definition(m, h, mask=None, S0=None, window=None):
    """The layer in float64 from its parameters (p: double leaves)."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in m.named_parameters()}
    lin = lambda n, x: x @ p[n + ".weight"].t() + (p[n + ".bias"] if n + ".bias" in p else 0)  # noqa: E731
    xz = lin("in_proj", h)
    x, z = xz[..., :m.inner], xz[..., m.inner:]
    x, win = ref.conv(x, p["conv_weight"], p.get("conv_bias"), "silu", mask, window)
    q = lin("x_proj", x)
    R, GN = m.dt_rank, m.groups * m.state_size
    B, C = (q[..., i:i + GN].unflatten(-1, (m.groups, m.state_size)) for i in (R, R + GN))
    y, S = ref.scan(x, lin("dt_proj", q[..., :R]), -torch.exp(p["A_log"]), B, C, p["D"], z, p["dt_bias"], True, mask, S0)
    return lin("out_proj", y), S, win, p


@pytest.mark.parametrize("groups,width,bias", [(1, 4, False), (2, 3, True)])
def test_layer_in_float32(groups, width, bias):
    m = layer(groups=groups, conv_width=width, bias=bias)
    h = torch.randn(2, 70, 48, device="cuda", requires_grad=True)
    mask = torch.ones(2, 70, dtype=torch.bool, device="cuda")
    mask[1, 50:] = False
    out, state = m(h, attention_mask=mask, use_cache=True)
    h64 = h.detach().double().requires_grad_(True)
    want, S, win, p = definition(m, h64, mask)
    assert rel(out, want) < 2e-5 and rel(state, S) < 2e-5 and rel(state.Z, win) < 2e-5
    g = torch.randn_like(out)
    out.backward(g)
    names = list(p)
    grads = torch.autograd.grad((want * g.double()).sum(), [h64] + [p[n] for n in names])
    assert rel(h.grad, grads[0]) < 2e-5
    for n, e in zip(names, grads[1:]):
        assert rel(dict(m.named_parameters())[n].grad, e) < 2e-5, n


def test_layer_under_autocast():
    m = layer(128)
    h = torch.randn(2, 90, 128, device="cuda", requires_grad=True)
    with torch.autocast("cuda", torch.bfloat16):
        out, _ = m(h)
    assert out.dtype == torch.bfloat16
    h64 = h.detach().double().requires_grad_(True)
    want, _, _, p = definition(m, h64)
    assert rel(out, want) < 3e-2
    g = torch.randn_like(out)
    out.backward(g)
    grads = dict(zip(p, torch.autograd.grad((want * g.double()).sum(), list(p.values()))))
    for n, e in grads.items():
        assert rel(dict(m.named_parameters())[n].grad, e) < 4e-2, n


def test_gradients_through_the_states():
    """Two pieces with the state handed on equal one pass, gradients too (they flow through both states)."""
    m = layer()
    h = torch.randn(2, 60, 48, device="cuda", requires_grad=True)
    out, _ = m(h)
    g = torch.randn_like(out)
    (whole,) = torch.autograd.grad(out, h, g, retain_graph=False)
    first, state = m(h[:, :23], use_cache=True)
    second, _ = m(h[:, 23:], past_state=state, use_cache=True)
    both = torch.cat([first, second], 1)
    assert rel(both, out) < 1e-5
    (parts,) = torch.autograd.grad(both, h, g)
    assert rel(parts, whole) < 2e-5


def test_generation_through_the_cache():
    """A padded batch of prompts, then single tokens through two blocks, beams reordered on the way."""
    torch.manual_seed(1)
    blocks = torch.nn.ModuleList([SubQStateSpaceBlock(64) for _ in range(2)]).cuda()
    last = SubQRMSNorm(64).cuda()
    x = torch.randn(3, 30, 64, device="cuda")
    lens = [30, 17, 0]
    with torch.no_grad():
        mask = torch.zeros(3, 30, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            mask[i, :n] = True
        cache = StateCache()
        _, states = run_layers(blocks, x, attention_mask=mask)
        cache.step(states, 30)
        new = torch.randn(3, 5, 64, device="cuda")
        got = []
        for t in range(5):
            pair, states = run_layers(blocks, new[:, t:t + 1], past_key_values=cache.to_legacy())
            cache.step(states, 1)
            got.append(last(*pair)[0])
        assert cache.get_seq_length() == 35 and cache.memory_bytes() == 2 * 3 * 128 * (16 + 3) * 4
        for i, n in enumerate(lens):
            pair, _ = run_layers(blocks, torch.cat([x[i:i + 1, :n], new[i:i + 1]], 1))
            assert rel(torch.cat(got, 1)[i:i + 1], last(*pair)[0][:, n:]) < 2e-5
        cache.reorder(torch.tensor([1, 1, 0]))
        pair, _ = run_layers(blocks, new[[1, 1, 0], :1], past_key_values=cache.to_legacy())
        pair1, _ = run_layers(blocks, torch.cat([x[1:2, :17], new[1:2], new[1:2, :1]], 1))
        assert rel(last(*pair)[0][:1], last(*pair1)[0][:, -1:]) < 2e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantised_blocks_serve(dtype):
    torch.manual_seed(2)
    blocks = torch.nn.ModuleList([SubQStateSpaceBlock(256) for _ in range(2)]).cuda()
    last = SubQRMSNorm(256).cuda()
    x = torch.randn(2, 40, 256, device="cuda", dtype=dtype)
    with torch.no_grad():
        want = last(*run_layers(blocks, x.float())[0])[0]
        for b in blocks:
            b.quantize()
            b.mixer.in_proj.out_dtype = dtype
        if dtype != torch.float32:
            blocks.to(dtype)
            assert isinstance(blocks[0].mixer.in_proj, SubQFp8Linear) and blocks[0].mixer.in_proj.scale_bytes.dtype == torch.uint8
        got, states = run_layers(blocks, x)
        assert rel(last(*got)[0], want) < 0.1 + (3e-2 if dtype != torch.float32 else 0)
        # pieces and steps equal one pass
        pair, st = run_layers(blocks, x[:, :39])
        pair, st = run_layers(blocks, x[:, 39:], past_key_values=st)
        assert rel(last(*pair)[0], last(*got)[0][:, 39:]) < (2e-2 if dtype == torch.float32 else 5e-2)  # (a rounding to 8 bits may differ)
    with pytest.raises(RuntimeError, match="inference"):
        blocks[0](x.requires_grad_(True))


def test_quantised_linear_against_its_own_weights():
    lin = torch.nn.Linear(200, 300).cuda()
    q = SubQFp8Linear.from_linear(lin)
    x = torch.randn(5, 7, 200, device="cuda")
    with torch.no_grad():
        got = q(x)
        a, sa = ops.quantize_fp8(x)
        w = q.weight_bytes.view(torch.float8_e4m3fn)[:, :200]
        want = ref.matmul(a, sa, w, q.scale_bytes.view(torch.float32), q.bias)
        assert rel(got, want) < 4e-6
        assert rel(got, lin(x)) < 6e-2
    copy = SubQFp8Linear(200, 300).cuda()
    copy.load_state_dict(q.state_dict())
    with torch.no_grad():
        assert torch.equal(copy(x), got)


def test_norm_gradients_with_the_stream():
    x = torch.randn(40, 100, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    s = torch.randn(40, 100, device="cuda", requires_grad=True)
    w = torch.randn(100, device="cuda", requires_grad=True)
    for only in ("both", "y", "r"):
        y, r = rms_norm(x, w, 1e-5, s)
        gy, gr = torch.randn_like(y), torch.randn_like(r)
        loss = (y * gy).sum().float() * (only != "r") + (r * gr).sum() * (only != "y")
        loss = (y * gy).float().sum() if only == "y" else (r * gr).sum() if only == "r" else (y * gy).float().sum() + (r * gr).sum()
        dx, ds, dw = torch.autograd.grad(loss, (x, s, w), allow_unused=True)
        leaf, wl = r.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
        want = 0
        if only != "r":
            want = want + (ref.rms(leaf, wl) * gy.double()).sum()
        if only != "y":
            want = want + (leaf * gr.double()).sum()
        e, ew = torch.autograd.grad(want, (leaf, wl), allow_unused=True)
        assert rel(ds, e) < 5e-6 and rel(dx, e) < 2.0 ** -8
        assert dx.dtype == torch.bfloat16 and ds.dtype == torch.float32
        if only != "r":
            assert rel(dw, ew) < 3e-6
    x32 = torch.randn(8, 64, device="cuda", requires_grad=True)
    y = rms_norm(x32, None, out_dtype=torch.bfloat16)
    (g,) = torch.autograd.grad(y.float().square().sum(), x32)
    assert g.dtype == torch.float32


def test_captured_training_step():
    """Forward and backward of the block in one graph, replayed on new inputs."""
    m = SubQStateSpaceBlock(64).cuda()
    x = torch.randn(2, 40, 64, device="cuda")
    params = list(m.parameters())

    def step():
        (out, stream), _ = m(x)
        return torch.autograd.grad((out.square().sum() + stream.sum()), params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    got = [g.clone() for g in held]
    for a, b in zip(got, step()):
        assert rel(a, b) < 1e-6


def test_checkpointing_and_compile():
    from torch.utils.checkpoint import checkpoint

    m = SubQStateSpaceBlock(64).cuda()
    x = torch.randn(2, 50, 64, device="cuda", requires_grad=True)
    want = torch.autograd.grad(m(x)[0][0].square().sum(), [x] + list(m.parameters()))
    got = torch.autograd.grad(checkpoint(lambda h: m(h)[0][0], x, use_reentrant=False).square().sum(), [x] + list(m.parameters()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    traced = torch.compile(lambda h: m(h)[0][0], fullgraph=True, backend="aot_eager")
    got = torch.autograd.grad(traced(x).square().sum(), [x] + list(m.parameters()))
    assert all(rel(a, b) < 1e-5 for a, b in zip(got, want))


def test_operators_have_schemas_and_fakes():
    t = ("test_schema", "test_faketensor")
    u = torch.randn(2, 12, 32, device="cuda")
    B = torch.randn(2, 12, 2, 8, device="cuda")
    A, D = -torch.rand(32, 8, device="cuda"), torch.ones(32, device="cuda")
    S = torch.randn(2, 32, 8, device="cuda")
    mask = torch.ones(2, 12, dtype=torch.uint8, device="cuda")
    o = torch.ops.subq_audio
    for more in ((D, u, D, mask, S), (None, None, None, None, None)):
        torch.library.opcheck(o.selective_scan_fwd, (u, u, A, B, B, *more, True, True, True), test_utils=t)
        h = o.selective_scan_fwd(u, u, A, B, B, *more, True, True, True)[2]
        torch.library.opcheck(o.selective_scan_bwd, (u, u, A, B, B, u, *more, more[4], True, h, more[4] is not None), test_utils=t)
    w, win = torch.randn(32, 4, device="cuda"), torch.randn(2, 3, 32, device="cuda")
    torch.library.opcheck(o.causal_conv_fwd, (u, w, D, mask, win, "silu", True), test_utils=t)
    torch.library.opcheck(o.causal_conv_fwd, (u, w, None, None, None, None, False), test_utils=t)
    torch.library.opcheck(o.causal_conv_bwd, (u, w, u, D, mask, win, win, "silu", True), test_utils=t)
    torch.library.opcheck(o.rms_norm_fwd, (u.half(), D, u, 1e-5, None), test_utils=t)
    torch.library.opcheck(o.rms_norm_fwd, (u, None, None, 1e-5, torch.bfloat16), test_utils=t)
    torch.library.opcheck(o.rms_norm_bwd, (u.half(), u, D, u, 1e-5, True), test_utils=t)
    torch.library.opcheck(o.rms_norm_bwd, (u, u, D, None, 1e-5, False), test_utils=t)


def test_second_gradients_and_bad_states_raise():
    u = torch.randn(1, 8, 16, device="cuda", requires_grad=True)
    B = torch.randn(1, 8, 4, device="cuda")
    y, _ = selective_scan(u, u, -torch.rand(16, 4, device="cuda"), B, B)
    (g,) = torch.autograd.grad(y.sum(), u, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), u)
    y, _ = causal_conv(u, torch.randn(16, 3, device="cuda"))
    (g,) = torch.autograd.grad(y.sum(), u, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), u)
    m = layer()
    with pytest.raises(ValueError, match="window"):
        m(torch.randn(1, 4, 48, device="cuda"), past_state=torch.zeros(1, 96, 16, device="cuda"))


def test_a_refused_call_leaves_nothing_behind():
    """Sizes that the library gave are kept by the calls' sizes; a refused call's answer (none) is not."""
    x = torch.randn(3, 77, 40, device="cuda")
    w = torch.randn(40, 4, device="cuda")
    for _ in range(2):
        with pytest.raises(ValueError):
            ops.causal_conv_backward(x, w, x[:, :76])
        with pytest.raises(ValueError):
            ops.selective_scan_backward(x, x, -torch.rand(40, 6, device="cuda"), x[..., :6], x[..., :6], x, z=x[:2])
        with pytest.raises(ValueError):
            ops.rms_norm_backward(x, x, w[:39, 0])
    assert ops.causal_conv_backward(x, w, x)[0].shape == x.shape
    assert ops.selective_scan_backward(x, x, -torch.rand(40, 6, device="cuda"), x[..., :6], x[..., :6], x).du.shape == x.shape


def test_inputs_on_a_side_stream_and_many_calls_at_once():
    """Calls of every operator on two streams at once, with their own workspaces."""
    torch.manual_seed(3)
    x = torch.randn(2, 600, 64, device="cuda", dtype=torch.bfloat16)
    A, B, w = -torch.rand(64, 16, device="cuda"), torch.randn(2, 600, 16, device="cuda", dtype=torch.bfloat16), torch.randn(64, 4, device="cuda")
    q = ops.quantize_fp8(x)
    qw = ops.quantize_fp8_weight(torch.randn(96, 64, device="cuda"))

    def everything():
        g = ops.selective_scan_backward(x, x, A, B, B, x)
        return (*(t for t in g if t is not None), *(t for t in ops.causal_conv_backward(x, w, x) if t is not None), *ops.rms_norm_backward(x, x),
                ops.scaled_matmul(*q, *qw))

    want = everything()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(everything())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
