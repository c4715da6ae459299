"""The 8-bit projection (ops.scaled_matmul) against its definition in float64.

Tolerances, relative in the 2-norm: half a step of the result's type, u = eps / 2; inside, products of two e4m3 values are exact,
the tensor core adds 128 of them in float32 (cut off rather than rounded: at most 128 x 2^-23 of the largest partial sum,
sqrt(128) x 2^-23 = 1.3e-6 in the mean square), then one rounding a block of 128: 4e-6 with the blocks' own.
"""
import pytest
import torch

import block_reference as ref
from subq_audio import ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IN = 4e-6


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else 0.0


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n, d = float(b.norm()), float((a - b).norm())
    return d / n if n > 0 else d


def operands(M, N, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    a, sa = ops.quantize_fp8((torch.randn(M, K, generator=g) * (0.2 + torch.rand(M, 1, generator=g))).cuda())
    b, sb = ops.quantize_fp8_weight((torch.randn(N, K, generator=g) * (0.2 + torch.rand(N, K, generator=g))).cuda())
    return a, sa, b, sb


@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 129), (2, 64, 16), (3, 1000, 777), (4, 40, 2000), (5, 129, 128), (8, 1025, 1024), (9, 33, 100), (16, 512, 640),
                                   (100, 130, 257), (128, 128, 128), (129, 257, 1000), (300, 96, 48), (1000, 4096, 512), (2500, 2000, 300), (333, 777, 3001)])
def test_products(M, N, K, out):
    a, sa, b, sb = operands(M, N, K)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(4)).cuda()
    for extra in (None, bias):
        got = ops.scaled_matmul(a, sa, b, sb, bias=extra, out_dtype=T[out])
        want = ref.matmul(a, sa, b, sb, extra)
        assert got.dtype == T[out] and rel(got, want) < IN + half(T[out])
    ops.check_device_status()


def test_every_row_and_column_is_its_own():
    """Small whole numbers with scales of one and powers of two: exact, so that a misplaced value shows."""
    g = torch.Generator().manual_seed(1)
    for M, N, K in ((200, 300, 300), (7, 300, 300), (64, 5000, 256), (20000, 130, 128)):
        a = torch.randint(-3, 4, (M, K), generator=g).float().cuda().to(torch.float8_e4m3fn)
        b = torch.randint(-3, 4, (N, K), generator=g).float().cuda().to(torch.float8_e4m3fn)
        sa = torch.exp2(torch.randint(-2, 3, (M, -(-K // 128)), generator=g).float()).cuda()
        sb = torch.exp2(torch.randint(-2, 3, (-(-N // 128), -(-K // 128)), generator=g).float()).cuda()
        got = ops.scaled_matmul(a, sa, b, sb, out_dtype=torch.float32)
        assert torch.equal(got.double(), ref.matmul(a, sa, b, sb))


def test_shapes_strides_and_out():
    a, sa, b, sb = operands(60, 200, 256)
    want = ops.scaled_matmul(a, sa, b, sb)
    got = ops.scaled_matmul(a.view(3, 20, 256), sa.view(3, 20, 2), b, sb)
    assert got.shape == (3, 20, 200) and torch.equal(got.view(60, 200), want)
    wide = torch.zeros(60, 300, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wide[:, 3:259] = a  # rows on no 16-byte boundary
    assert torch.equal(ops.scaled_matmul(wide[:, 3:259], sa, b, sb), want)
    assert torch.equal(ops.scaled_matmul(a, sa.t().contiguous().t(), b, sb.t().contiguous().t()), want)
    out = torch.full((60, 203), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.scaled_matmul(a, sa, b, sb, out=out[:, :200])
    assert torch.equal(out[:, :200], want) and bool((out[:, 200:] == 7).all())
    assert ops.scaled_matmul(a[:0], sa[:0], b, sb).shape == (0, 200)
    none = ops.scaled_matmul(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0], bias=torch.arange(200.0, device="cuda"), out_dtype=torch.float32)
    assert torch.equal(none, torch.arange(200.0, device="cuda").expand(60, 200))


def test_nan_stays_in_its_row_and_graphs():
    a, sa, b, sb = operands(150, 140, 384)
    sa[3, 1] = float("nan")
    got = ops.scaled_matmul(a, sa, b, sb, out_dtype=torch.float32)
    assert bool(torch.isnan(got[3]).all()) and not bool(torch.isnan(got[4:]).any()) and not bool(torch.isnan(got[:3]).any())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.scaled_matmul(a, sa, b, sb, out_dtype=torch.float32)
    graph.replay()
    assert torch.equal(held.nan_to_num(5.0), got.nan_to_num(5.0))


def test_refusals():
    a, sa, b, sb = operands(20, 30, 200)
    with pytest.raises(TypeError):
        ops.scaled_matmul(a.float(), sa, b, sb)
    with pytest.raises(TypeError):
        ops.scaled_matmul(a, sa.double(), b, sb)
    with pytest.raises(TypeError):
        ops.scaled_matmul(a, sa, b, sb, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.scaled_matmul(a[:, :100], sa, b, sb)
    with pytest.raises(ValueError):
        ops.scaled_matmul(a, sa[:, :1], b, sb)
    with pytest.raises(ValueError):
        ops.scaled_matmul(a, sa, b, sb, out=torch.empty(20, 31, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        ops.scaled_matmul(a, sa, b, sb, out=torch.empty(1, 30, dtype=torch.bfloat16, device="cuda").expand(20, 30))
    with pytest.raises(RuntimeError):
        ops.scaled_matmul(a.cpu(), sa, b, sb)
