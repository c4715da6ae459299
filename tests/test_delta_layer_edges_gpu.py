"""SubQLayerNorm and SubQGatedDeltaAttention at the edges of what they stand in for."""
import pytest
import torch

from subq_audio import SubQLayerNorm
from test_delta_layer_gpu import Block, plain_block, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_refuses_another_width_as_torch_does(affine):
    for norm in (torch.nn.LayerNorm(64, elementwise_affine=affine).cuda(), SubQLayerNorm(64, elementwise_affine=affine).cuda()):
        for shape in ((3, 32), (3, 128), (64, 3), (2, 1)):
            with pytest.raises((RuntimeError, ValueError)):
                norm(torch.randn(*shape, device="cuda"))
        assert norm(torch.randn(5, 64, device="cuda")).shape == (5, 64)


@pytest.mark.parametrize("small", [1.0, 1e-3])
def test_heads_of_every_width_scale_queries_and_keys_alike(small):
    """x / sqrt(|x|^2 + 1e-6), by the norm's kernel (64) and without it (80): also where |x| is near the root of 1e-6."""
    for d in (64, 80):
        torch.manual_seed(d)
        m = Block(d=2 * d, heads=2, kv=1).cuda()
        with torch.no_grad():
            m.attn.q_proj.weight.mul_(small)
            m.attn.k_proj.weight.mul_(small)
        x = torch.randn(2, 70, 2 * d, device="cuda", requires_grad=True)
        w = torch.randn(2, 70, 2 * d, device="cuda")
        got = torch.autograd.grad((m(x)[0] * w).sum(), [x, *m.parameters()])
        x64 = x.detach().double().requires_grad_(True)
        y64, p = plain_block(m, x64)
        want = torch.autograd.grad((y64 * w.double()).sum(), [x64, *p.values()])
        # the tolerances of test_delta_layer_gpu.py's float32 block
        assert rel(m(x)[0], y64) < 1e-5
        for (n, _), a, b in zip([("x", x), *m.named_parameters()], got, want):
            assert rel(a, b) < 3e-5, (d, n)


def test_layer_norm_keeps_float32_under_autocast_where_it_is_asked_to():
    torch.manual_seed(3)
    x = torch.randn(7, 96, device="cuda", requires_grad=True)
    plain, norm = torch.nn.LayerNorm(96).cuda(), SubQLayerNorm(96, out_dtype=torch.float32).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want, got, default = plain(x), norm(x), SubQLayerNorm(96).cuda()(x)
    assert want.dtype == got.dtype == torch.float32 and default.dtype == torch.bfloat16
    assert rel(got, want) < 1e-6  # float32 sums of 96 terms on both sides (test_layer_norm_gpu.py)
    w = torch.randn_like(want)
    assert rel(torch.autograd.grad((got * w).sum(), x)[0], torch.autograd.grad((want * w).sum(), x)[0]) < 2e-6
    assert SubQLayerNorm(96, out_dtype=torch.float16).cuda()(x).dtype == torch.float16
    assert norm(x.half()).dtype == torch.float16


def test_what_layer_norm_does_not_differentiate_raises():
    x = torch.randn(3, 96, device="cuda", requires_grad=True)
    norm = SubQLayerNorm(96).cuda()
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: norm(t).square().sum())(x.detach())
    with pytest.raises(RuntimeError):
        torch.func.jvp(norm, (x.detach(),), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(norm(x).square().sum(), x, create_graph=True)[0].sum().backward()


def test_checkpointed_layer_and_inference_mode():
    """Under torch.utils.checkpoint the forward's handover is not kept until the backward; the gradients are the same."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(6)
    m = Block().cuda()
    x = torch.randn(4, 2048, 256, device="cuda", requires_grad=True)
    params = [x, *m.parameters()]

    def run(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = call(x)
        held = torch.cuda.memory_allocated() - before
        return held, torch.autograd.grad(y.square().mean(), params)

    whole, want = run(lambda t: m(t)[0])
    less, got = run(lambda t: checkpoint(lambda u: m(u)[0], t, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    handover = 4 * 4 * (2048 // 64) * 79 * 1024  # of 4 x 4 heads of 32 chunks
    assert whole > handover and less < whole - handover
    with torch.inference_mode():
        assert torch.equal(m(x)[0], m(x.detach())[0])
