"""The gated-delta layer and the layer norm before it, used together as a model
uses them: the operators' schemas and fake kernels, the differentiable calls
against float64 autograd, a block (norm, layer, residual) in training, prompt
then single tokens through the per-layer cache, padding, and tracing.

Tolerances: test_delta_gpu.py derives the kernels' own; a float32 block of a
few products of 128 terms on top stays within 1e-5, a bf16 one within a few
roundings of 2^-8 each (2e-2).
"""
import pytest
import torch
import torch.nn.functional as F

import delta_reference as ref
from subq_audio import SubQGatedDeltaAttention, SubQLayerNorm, gated_delta_attention, layer_norm, ops
from subq_audio.cache import StateCache, run_layers

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    assert a.shape == b.shape
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def inputs(B=2, H=4, Hkv=2, N=150, d=64, e=64, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = F.normalize(torch.randn(B, N, H, d, generator=g), dim=-1).to(dtype).cuda().transpose(1, 2)
    k = F.normalize(torch.randn(B, N, Hkv, d, generator=g), dim=-1).to(dtype).cuda().transpose(1, 2)
    v = torch.randn(B, N, Hkv, e, generator=g).to(dtype).cuda().transpose(1, 2)
    beta = torch.sigmoid(torch.randn(B, H, N, generator=g)).cuda()
    lg = -F.softplus(-(torch.randn(B, H, N, generator=g) + 2)).cuda()
    S0 = 0.3 * torch.randn(B, H, d, e, generator=g).cuda()
    return q, k, v, beta, lg, S0


@pytest.mark.parametrize("gates", ["token", "head", "scalar", "none"])
def test_autograd_against_float64(gates):
    q, k, v, beta, lg, S0 = inputs()
    B, H, N = beta.shape
    if gates == "head":
        beta, lg = beta[0, :, 0].clone(), lg[0, :, 0].clone()
    elif gates == "scalar":
        beta, lg = beta[0, 0, 0].clone(), lg[0, 0, 0].clone()
    mask = torch.ones(B, N, dtype=torch.bool, device="cuda")
    mask[1, 100:] = False
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    leaves += [] if gates == "none" else [beta.requires_grad_(True), lg.requires_grad_(True)]
    leaves.append(S0.requires_grad_(True))
    b_, l_ = (None, None) if gates == "none" else leaves[3:5]
    out, S = gated_delta_attention(leaves[0], leaves[1], leaves[2], b_, l_, S0, mask)
    w, wS = torch.randn_like(out), torch.randn_like(S)
    got = torch.autograd.grad((out * w).sum() + (S * wS).sum(), leaves)
    lv = [x.detach().double().requires_grad_(True) for x in leaves]

    def full(x, other):
        if x is None:
            return torch.full((B, H, N), other, dtype=torch.float64, device="cuda")
        return (x.view(1, -1, 1) if x.dim() == 1 else x).expand(B, H, N)

    rb, rl = (None, None) if gates == "none" else lv[3:5]
    fb, fl = full(rb, 1.0), full(rl, 0.0)
    if gates == "none":
        fb.requires_grad_(True), fl.requires_grad_(True)
    ro, rS = ref.rule(lv[0], lv[1], lv[2], fb, fl, mask, 64 ** -0.5, lv[-1])
    want = torch.autograd.grad((ro * w.double()).sum() + (rS * wS.double()).sum(), lv + [fb, fl])
    assert rel(out, ro) < 6e-6 and rel(S, rS) < 6e-6
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.shape == b.shape
        if i in (3, 4) and gates in ("head", "scalar"):
            # a sum of n per-token gradients, each off by 1e-5 of their root mean square, is off by sqrt(n) times that,
            # which is 1e-5 of their 2-norm, whatever is left of the sum itself; for log gamma the 64 tokens of a chunk
            # share the error of the chunk's end term and of the suffix sums, so their errors add up as they are: 64
            # in place of sqrt(64), 8 times as much
            assert float((a.double() - b).norm()) < (8e-5 if i == 4 else 1e-5) * float(want[len(lv) + i - 3].norm()), i
        else:
            assert rel(a, b) < 1e-5, i


def test_only_the_state_and_3d_inputs():
    q, k, v, beta, lg, S0 = inputs(H=1, Hkv=1)
    q, k, v, beta, lg = (x[:, 0].contiguous().requires_grad_(True) for x in (q, k, v, beta, lg))
    out, S = gated_delta_attention(q, k, v, beta, lg)
    assert out.shape == v.shape
    g = torch.autograd.grad(S.square().sum(), (k, v, beta, lg))
    k2, v2, b2, l2 = (x.detach().double().unsqueeze(1).requires_grad_(True) for x in (k, v, beta, lg))
    _, rS = ref.rule(q.detach().double().unsqueeze(1), k2, v2, b2, l2, None, 1.0, torch.zeros(2, 1, 64, 64, device="cuda").double())
    want = torch.autograd.grad(rS.square().sum(), (k2, v2, b2, l2))
    for a, b in zip(g, want):
        assert rel(a, b.squeeze(1)) < 1e-5
    with pytest.raises(RuntimeError, match="once_differentiable"):
        o, _ = gated_delta_attention(q, k, v, beta, lg)
        (d,) = torch.autograd.grad(o.square().sum(), q, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operators_schema_and_fake_kernels(dtype):
    q, k, v, beta, lg, S0 = inputs(dtype=dtype)
    check = dict(test_utils=("test_schema", "test_faketensor"))
    fwd = (q, k, v, beta, lg, None, S0, 0.125, True, True)
    torch.library.opcheck(torch.ops.subq_audio.gated_delta_fwd.default, fwd, **check)
    o, S, handover = torch.ops.subq_audio.gated_delta_fwd(*fwd)
    torch.library.opcheck(torch.ops.subq_audio.gated_delta_bwd.default,
                          (q, k, v, beta, torch.randn_like(o), lg, None, S0, torch.randn_like(S), 0.125, handover, True, True), **check)
    x = torch.randn(3, 40, 96, device="cuda", dtype=dtype)
    w = torch.rand(96, device="cuda")
    torch.library.opcheck(torch.ops.subq_audio.layer_norm_fwd.default, (x, w, w, 1e-5, torch.bfloat16), **check)
    torch.library.opcheck(torch.ops.subq_audio.layer_norm_bwd.default, (torch.randn_like(x), x, w, 1e-5, True, False), **check)


def test_layer_norm_module_equals_torch():
    torch.manual_seed(0)
    a, b = SubQLayerNorm(96).cuda(), torch.nn.LayerNorm(96).cuda()
    b.load_state_dict(a.state_dict())
    x = torch.randn(5, 33, 96, device="cuda", requires_grad=True)
    w = torch.randn(5, 33, 96, device="cuda")
    ga = torch.autograd.grad((a(x) * w).sum(), [x, *a.parameters()])
    gb = torch.autograd.grad((b(x) * w).sum(), [x, *b.parameters()])
    assert all(rel(p, q) < 2e-6 for p, q in zip(ga, gb))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = a(x)
        assert y.dtype == torch.bfloat16 and rel(y, b(x)) < 2.0 ** -8
    assert layer_norm(x.detach()).shape == x.shape


class Block(torch.nn.Module):
    def __init__(self, d=256, heads=4, kv=2):
        super().__init__()
        self.ln, self.attn = SubQLayerNorm(d), SubQGatedDeltaAttention(d, heads, kv)

    def forward(self, x, past_state=None, attention_mask=None, use_cache=False):
        y, state = self.attn(self.ln(x), past_state=past_state, attention_mask=attention_mask, use_cache=use_cache)
        return x + y, state


def plain_block(m, x, mask=None):
    """The block in float64 torch operations."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in m.named_parameters()}
    h = F.layer_norm(x, x.shape[-1:], p["ln.weight"], p["ln.bias"], m.ln.eps)
    B, L, D = h.shape
    a = m.attn

    def heads(n):
        return (h @ p[f"attn.{n}.weight"].T).view(B, L, -1, a.head_dim).transpose(1, 2)

    def unit(t):  # (as the kernel's eps has it)
        return t * torch.rsqrt(t.square().sum(-1, keepdim=True) + 1e-6)

    beta = torch.sigmoid(h @ p["attn.beta_proj.weight"].T).transpose(1, 2)
    lg = -F.softplus(-(p["attn.raw_decay"] + h @ p["attn.gate_proj.weight"].T)).transpose(1, 2)
    o, _ = ref.rule(unit(heads("q_proj")), unit(heads("k_proj")), heads("v_proj"), beta, lg, mask, 1.0,
                    torch.zeros(B, a.num_heads, a.head_dim, a.head_dim, dtype=torch.float64, device=x.device))
    o = F.rms_norm(o, (a.head_dim,), p["attn.head_norm.weight"], a.head_norm.eps)
    return x + o.transpose(1, 2).reshape(B, L, D) @ p["attn.out_proj.weight"].T, p


def test_block_training_against_float64():
    torch.manual_seed(1)
    m = Block().cuda()
    x = torch.randn(2, 130, 256, device="cuda", requires_grad=True)
    mask = torch.ones(2, 130, dtype=torch.bool, device="cuda")
    mask[0, 90:] = False
    y, _ = m(x, attention_mask=mask)
    w = torch.randn_like(y)
    got = torch.autograd.grad((y * w).sum(), [x, *m.parameters()])
    x64 = x.detach().double().requires_grad_(True)
    y64, p = plain_block(m, x64, mask)
    want = torch.autograd.grad((y64 * w.double()).sum(), [x64, *p.values()])
    assert rel(y, y64) < 1e-5
    for (n, _), a, b in zip([("x", x), *m.named_parameters()], got, want):
        assert rel(a, b) < 3e-5, n
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y16, _ = m(x, attention_mask=mask)
    assert rel(y16, y64) < 2e-2
    g16 = torch.autograd.grad((y16 * w).sum(), [x, *m.parameters()])
    assert all(torch.isfinite(t).all() for t in g16) and rel(g16[0], want[0]) < 3e-2


def test_prompt_then_tokens_through_the_cache():
    """run_layers and StateCache with these layers: a prompt in one pass, then single tokens, equal one pass over all;
    reordering the batch (beam search) reorders the states."""
    torch.manual_seed(2)
    layers = torch.nn.ModuleList([Block(), Block()]).cuda().eval()
    x = torch.randn(3, 90, 256, device="cuda")
    with torch.no_grad():
        whole, states = run_layers(layers, x)
        y, past = run_layers(layers, x[:, :83])
        cache = StateCache()
        cache.step(past, 83)
        outs = [y]
        for t in range(83, 90):
            y, past = run_layers(layers, x[:, t:t + 1], past_key_values=cache.to_legacy())
            cache.step(past, 1)
            outs.append(y)
        assert rel(torch.cat(outs, 1), whole) < 1e-5
        assert all(rel(a, b) < 1e-5 for a, b in zip(cache.to_legacy(), states))
        assert cache.get_seq_length() == 90 and cache.memory_bytes() == 2 * 3 * 4 * 64 * 64 * 4
        order = torch.tensor([2, 0, 0], device="cuda")
        cache.reorder(order)
        y2, _ = run_layers(layers, x[order, 89:90], past_key_values=cache.to_legacy())
        y1, _ = run_layers(layers, x[:, 89:90], past_key_values=states)
        assert rel(y2, y1[order]) < 1e-5


def test_layer_traces_with_fullgraph():
    torch.manual_seed(3)
    m = Block().cuda()
    x = torch.randn(2, 100, 256, device="cuda", requires_grad=True)
    ref_g = torch.autograd.grad(m(x)[0].square().mean(), [x, *m.parameters()])
    compiled = torch.compile(m, fullgraph=True, backend="aot_eager")
    y = compiled(x)[0]
    got = torch.autograd.grad(y.square().mean(), [x, *m.parameters()])
    torch.testing.assert_close(y, m(x)[0])
    for a, b in zip(got, ref_g):
        torch.testing.assert_close(a, b)


def test_captured_layer_step():
    """Forward and backward of a block captured in one CUDA graph and replayed on new inputs."""
    torch.manual_seed(4)
    m = Block().cuda()
    fixed = torch.randn(2, 100, 256, device="cuda", requires_grad=True)
    params = list(m.parameters())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(m(fixed)[0].square().mean(), [fixed, *params])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(m(fixed)[0].square().mean(), [fixed, *params])
    new = torch.randn(2, 100, 256, device="cuda")
    with torch.no_grad():
        fixed.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    held = [t.clone() for t in held]
    want = torch.autograd.grad(m(fixed)[0].square().mean(), [fixed, *params])
    assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_refusals():
    with pytest.raises(ValueError, match="divisible"):
        SubQGatedDeltaAttention(100, 3)
    with pytest.raises(ValueError, match="divisible"):
        SubQGatedDeltaAttention(128, 4, 3)
    q, k, v, beta, lg, S0 = inputs(d=160)
    q.requires_grad_(True)
    out, _ = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg)  # d > 128: the token-recurrent forward
    assert out.shape == (2, 4, 150, 64)
    with pytest.raises(RuntimeError, match="head_dim"):  # but no backward
        gated_delta_attention(q, k, v, beta, lg)[0].sum().backward()
