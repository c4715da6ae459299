"""The residual RMSNorm (ops.rms_norm, rms_norm_backward), its 8-bit output and the quantising calls against float64.

Tolerances. A value rounded once is off by at most half a step, u = eps / 2. Inside: a float32 sum of D squares over 32 or
more lanes (at most D / 32 + 16 roundings, halved by the root) and four products, below 40 x 2^-24 = 2.4e-6 at D = 2048
in the worst case and 16 x 2^-24 = 1e-6 in the mean square, in which the tensors are compared (2-norm). dweight sums the
rows, at most 2^11 here: 2e-6. An 8-bit value may be rounded to the other side where y / scale lies within the 2^-21 or so that
float32 leaves of a border between two values: fewer than one in 10^5, each by one step, at most 1/8 of it.
"""
import pytest
import torch

import block_reference as ref
from subq_audio import ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IN, SUM = 1e-6, 2e-6


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else 0.0


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n, d = float(b.norm()), float((a - b).norm())
    return d / n if n > 0 else d


def rows(shape, dtype, seed, layout="plain"):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * (0.5 + torch.rand(shape[-1], generator=torch.Generator().manual_seed(seed + 1)))
    x = x.to(T[dtype])
    if layout == "odd":
        wide = torch.zeros(*shape[:-1], shape[-1] + 3, dtype=T[dtype])
        wide[..., 1:-2] = x
        return wide.cuda()[..., 1:-2]
    return x.cuda()


WIDTHS = [1, 7, 8, 64, 127, 128, 129, 250, 256, 500, 768, 1000, 1024, 1500, 2048, 4000, 8192, 10001, 16384]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("x_type,r_type", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_norm_with_residual(D, x_type, r_type):
    n = 37
    x, res, dr = rows((n, D), x_type, 0), rows((n, D), r_type, 2), rows((n, D), r_type, 4)
    w = (1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(6))).cuda()
    dy = rows((n, D), x_type, 8)
    y, r = ops.rms_norm(x, w, 1e-5, residual=res)
    assert r.dtype == T[r_type] and torch.equal(r, (x.float() + res.float()).to(T[r_type]))
    leaf, wl = r.double().requires_grad_(True), w.double().requires_grad_(True)
    want = ref.rms(leaf, wl)
    assert y.dtype == T[x_type] and rel(y, want.detach()) < IN + half(T[x_type])
    g, gw = torch.autograd.grad((want * dy.double()).sum() + (leaf * dr.double()).sum(), (leaf, wl))
    dx, dres, dw = ops.rms_norm_backward(dy, r, w, 1e-5, dresidual=dr)
    # (the norm's own part may cancel against dr: errors are relative to the terms)
    size = float(g.norm()) + float(dr.double().norm())
    for a in (dx, dres):
        assert float((a.double() - g).norm()) < (2 * IN + half(a.dtype)) * size
    assert rel(dw, gw) < SUM
    assert dx.dtype == T[x_type] and dres.dtype == T[r_type]


@pytest.mark.parametrize("D", [5, 96, 129, 1024, 3000])
@pytest.mark.parametrize("out", ["fp32", "bf16", "fp16"])
def test_norm_alone_and_types(D, out):
    x = rows((3, 11, D), "fp32", 1, "odd")
    y = ops.rms_norm(x, None, 1e-6, out_dtype=T[out])
    assert y.is_contiguous() and rel(y, ref.rms(x.double(), None, 1e-6)) < IN + half(T[out])
    dx, dres, dw = ops.rms_norm_backward(rows((3, 11, D), "fp32", 3), x, None, 1e-6, need_dweight=False)
    assert dx is dres and dw is None
    leaf = x.double().requires_grad_(True)
    (g,) = torch.autograd.grad((ref.rms(leaf, None, 1e-6) * rows((3, 11, D), "fp32", 3).double()).sum(), leaf)
    assert float((dx.double() - g).norm()) < 2 * IN * max(float(g.norm()), float(rows((3, 11, D), "fp32", 3).double().norm() / 8))


def check_fp8(q, scale, y, what):
    want_q, want_scale = ref.quantize(y)
    assert q.dtype == torch.float8_e4m3fn and rel(scale, want_scale) < IN, what
    d = (q.double() - want_q).abs()
    off = d > 0
    assert float(off.double().mean()) < 1e-5 + 1.5 / q.numel(), what
    assert bool((d <= want_q.abs() / 8 + 2.0 ** -9).all()), what


@pytest.mark.parametrize("D", [1, 16, 100, 128, 130, 768, 1000, 1024, 2049, 8192, 16384])
@pytest.mark.parametrize("x_type,r_type", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
def test_norm_to_8_bits(D, x_type, r_type):
    n = 61
    x, res = rows((n, D), x_type, 0), rows((n, D), r_type, 2)
    w = (1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(6))).cuda()
    q, scale, r = ops.rms_norm_fp8(x, w, 1e-5, residual=res)
    assert torch.equal(r, (x.float() + res.float()).to(T[r_type])) and scale.shape == (n, -(-D // 128))
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    check_fp8(q, scale, ref.rms(r.double(), w.double()), "norm")
    q, scale = ops.rms_norm_fp8(x, w, 1e-5)
    check_fp8(q, scale, ref.rms(x.double(), w.double()), "alone")
    q, scale = ops.quantize_fp8(x)
    check_fp8(q, scale, x.double(), "quantize")


def test_eight_bits_at_the_borders():
    """Zero rows, blocks below the floor, large and tiny values, infinities and NaN."""
    x = torch.zeros(7, 300, device="cuda")
    x[1] = 1e-38
    x[2] = 3e38
    x[3, ::2] = -2.0
    x[4] = torch.linspace(-448, 448, 300, device="cuda")
    q, scale = ops.quantize_fp8(x)
    want_q, want_scale = ref.quantize(x.double())
    assert torch.equal(q.double()[:5], want_q[:5]) and rel(scale[:5], want_scale[:5]) < IN
    x[5, 7], x[6, 200] = float("nan"), float("inf")
    q, scale = ops.quantize_fp8(x)
    assert bool(torch.isnan(scale[5, 0])) and bool(torch.isnan(q[5, :128].float()).all()) and not bool(torch.isnan(q[5, 128:].float()).any())
    assert bool(torch.isinf(scale[6, 1])) and not bool(torch.isnan(q[6, :128].float()).any())
    y, r = ops.rms_norm(x, residual=torch.zeros_like(x))
    assert bool(torch.isnan(y[5]).all()) and float(y[0].abs().max()) == 0
    # every half-way value between two neighbours of one binade goes to the even one
    mids = torch.tensor([(16 + 2 * i + 1) / 2 for i in range(8)], device="cuda")  # 8.5 .. 15.5, between integers
    row = torch.cat([mids, torch.full((120,), 448.0, device="cuda")])[None]
    q, scale = ops.quantize_fp8(row)
    assert float(scale) == 1.0 and torch.equal(q[0, :8].float(), ref.to_e4m3(mids.double()).float())


def test_weights_in_8_bits():
    g = torch.Generator().manual_seed(0)
    for N, K in ((1, 1), (130, 200), (256, 384)):
        w = torch.randn(N, K, generator=g).cuda()
        q, scale = ops.quantize_fp8_weight(w)
        assert q.shape == (N, K) and q.stride(0) % 16 == 0 and scale.shape == (-(-N // 128), -(-K // 128))
        back = q.double() * scale.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
        top = scale.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K] * 2.0 ** -10
        assert bool(((back - w.double()).abs() <= w.double().abs() / 16 * (1 + 1e-6) + top).all())


def test_in_place_views_streams_and_repeats():
    x, res = rows((40, 768), "bf16", 0, "odd"), rows((40, 768), "fp32", 2, "odd")
    want = ops.rms_norm(x.contiguous(), None, residual=res.contiguous())
    got = ops.rms_norm(x, None, residual=res)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    t = rows((6, 20, 768), "bf16", 0).transpose(0, 1)  # leading dimensions that do not merge
    assert torch.equal(ops.rms_norm(t), ops.rms_norm(t.contiguous()))
    dy = rows((5000, 768), "bf16", 3)
    r = rows((5000, 768), "fp32", 5)
    first, second = (ops.rms_norm_backward(dy, r) for _ in range(2))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.rms_norm_backward(dy, r)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, held))


def test_no_rows():
    x = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16)
    y, r = ops.rms_norm(x, residual=x)
    assert y.shape == (0, 64) and r.shape == (0, 64)
    q, s = ops.rms_norm_fp8(x)
    assert q.shape == (0, 64) and s.shape == (0, 1)
    _, _, dw = ops.rms_norm_backward(x, x)
    assert float(dw.abs().max()) == 0


def test_refusals():
    x = rows((4, 64), "bf16", 0)
    with pytest.raises(RuntimeError):
        ops.rms_norm(x.cpu())
    with pytest.raises(ValueError):
        ops.rms_norm(torch.zeros(2, 16385, device="cuda"))
    with pytest.raises(TypeError):
        ops.rms_norm(x.double())
    with pytest.raises(TypeError):
        ops.rms_norm(x, out_dtype=torch.float16)
    with pytest.raises(TypeError):
        ops.rms_norm(x, residual=x.half())
    with pytest.raises(ValueError):
        ops.rms_norm(x, residual=x[:2])
    with pytest.raises(ValueError):
        ops.rms_norm(x, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError):
        ops.rms_norm_backward(x, x[:2])
    with pytest.raises(ValueError):
        ops.rms_norm_backward(x, x, dresidual=x.float())
