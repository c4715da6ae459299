"""ops.layer_norm and ops.layer_norm_backward against layer norm in float64.

Tolerances, relative in the 2-norm: one rounding to the output's type (eps / 2;
none counted for float32) and float32 sums over D or over the rows inside. A sum
of n values in registers and a tree of partial sums is off by at most about
sqrt(n) 2^-24 of the values' norm in the mean square: below 1e-6 for a row (its
mean removed) and 3e-6 for column sums of 10^5 rows.
"""
import pytest
import torch

from subq_audio import _capi, ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n, d = float(b.norm()), float((a - b).norm())
    return d / n if n > 0 else d


def tol(dtype):
    return 1e-6 + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def reference(x, w, b, eps, dy=None):
    x, D = x.double(), x.shape[-1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    xc = x - x.mean(-1, keepdim=True)
    r = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = xc * r
    y = xh * w + (0 if b is None else b.double())
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, dx, (dy * xh).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)


def make(shape, x, y, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    D = shape[-1]
    v = torch.randn(*shape, generator=g, device="cuda") * (0.3 + torch.rand(D, generator=g, device="cuda")) + 0.5
    w, b = 1 + 0.3 * torch.randn(D, generator=g, device="cuda"), torch.randn(D, generator=g, device="cuda")
    return v.to(T[x]), w, b, torch.randn(*shape, generator=g, device="cuda").to(T[y])


PAIRS = [("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")]
SHAPES = [(1, 768), (3, 8), (1000, 64), (257, 256), (77, 264), (130, 1024), (33, 1032), (19, 4096), (9, 8192), (5, 8200),
          (40, 1), (31, 7), (12, 1021), (11, 1025), (7, 8191), (3, 20001), (2, 5, 3, 96)]


@pytest.mark.parametrize("x,y", PAIRS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_float64(shape, x, y):
    v, w, b, dy = make(shape, x, y, seed=shape[-1])
    ry, rdx, rdw, rdb = reference(v, w, b, 1e-5, dy)
    out = ops.layer_norm(v, w, b, 1e-5, out_dtype=T[y])
    assert out.dtype == T[y]
    if shape[-1] == 1:  # xh = 0: y is the bias, dx and dw are 0
        assert torch.equal(out.float(), b.to(T[y]).float().expand_as(out))
    else:
        assert rel(out, ry) < tol(T[y])
    dx, dw, db = ops.layer_norm_backward(dy, v, w, 1e-5)
    assert dx.dtype == T[x] and dw.dtype == db.dtype == torch.float32
    assert rel(dx, rdx) < tol(T[x])
    assert rel(dw, rdw) < 3e-6 and rel(db, rdb) < 3e-6
    again = ops.layer_norm_backward(dy, v, w, 1e-5)
    assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), again))


def test_many_rows_and_parts_not_wanted():
    v, w, b, dy = make((70001, 200), "fp32", "bf16")
    _, rdx, rdw, rdb = reference(v, w, b, 1e-5, dy)
    dx, dw, db = ops.layer_norm_backward(dy, v, w)
    assert rel(dx, rdx) < 1e-6 and rel(dw, rdw) < 3e-6 and rel(db, rdb) < 3e-6
    dx2, none, db2 = ops.layer_norm_backward(dy, v, w, need_dweight=False)
    assert none is None and torch.equal(dx2, dx) and torch.equal(db2, db)
    dx3, n1, n2 = ops.layer_norm_backward(dy, v, w, need_dweight=False, need_dbias=False)
    assert n1 is None and n2 is None and torch.equal(dx3, dx)


def test_no_weight_no_bias_and_strided_rows():
    v, _, _, dy = make((6, 50, 96), "bf16", "bf16")
    y = ops.layer_norm(v)
    assert rel(y, reference(v, None, None, 1e-5)) < tol(torch.bfloat16)
    wide = torch.randn(300, 200, device="cuda")
    for view in (wide[:, :96], wide[:, 4:100], wide[:, 1:97], wide[::3, :96], wide.t()):
        d = torch.randn(view.shape, device="cuda")
        y = ops.layer_norm(view)
        assert rel(y, reference(view, None, None, 1e-5)) < 1e-6
        dx, dw, db = ops.layer_norm_backward(d, view)
        _, rdx, rdw, rdb = reference(view, None, None, 1e-5, d)
        assert rel(dx, rdx) < 1e-6 and rel(dw, rdw) < 3e-6 and rel(db, rdb) < 3e-6
    half = torch.nn.LayerNorm(96).cuda().bfloat16()  # parameters in 16 bits are read in float32
    y = ops.layer_norm(v, half.weight, half.bias)
    assert rel(y, reference(v, half.weight, half.bias, 1e-5)) < tol(torch.bfloat16)


def test_constant_rows_large_offsets_and_no_rows():
    """A constant row has xh = 0 (its variance is exactly 0: the mean of equal values is exact up to
    rounding 2^-24 of it, far below sqrt(eps)); an offset of 1000 leaves float32's 2^-24 x 1000 of each
    value, 6e-5 of unit spread at most."""
    x = torch.full((4, 768), 3.0, device="cuda")
    b = torch.randn(768, device="cuda")
    y = ops.layer_norm(x, None, b)
    assert float((y - b).abs().max()) < 1e-3
    z = torch.randn(64, 768, device="cuda", dtype=torch.float64)
    y = ops.layer_norm((z + 1000).float())
    assert rel(y, reference((z + 1000).float(), None, None, 1e-5)) < 1e-4
    e = torch.empty(0, 3, 64, device="cuda")
    dx, dw, db = ops.layer_norm_backward(e, e, torch.ones(64, device="cuda"))
    assert ops.layer_norm(e).shape == e.shape and dx.shape == e.shape
    assert bool((dw == 0).all() and (db == 0).all())


def test_nan_row_stays_in_its_row():
    v, w, b, _ = make((9, 768), "fp32", "bf16")
    y = ops.layer_norm(v, w, b, out_dtype=torch.bfloat16)
    v[4, 5] = float("nan")
    z = ops.layer_norm(v, w, b, out_dtype=torch.bfloat16)
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(y[keep], z[keep]) and bool(z[4].isnan().all())


def test_captured_and_on_another_stream():
    v, w, b, dy = make((500, 768), "fp32", "bf16")
    want = (ops.layer_norm(v, w, b, out_dtype=torch.bfloat16),) + ops.layer_norm_backward(dy, v, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    fixed, fdy = torch.zeros_like(v), torch.zeros_like(dy)
    with torch.cuda.graph(graph):
        held = (ops.layer_norm(fixed, w, b, out_dtype=torch.bfloat16),) + ops.layer_norm_backward(fdy, fixed, w)
    fixed.copy_(v)
    fdy.copy_(dy)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = (ops.layer_norm(v, w, b, out_dtype=torch.bfloat16),) + ops.layer_norm_backward(dy, v, w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(held, want)) and all(torch.equal(a, c) for a, c in zip(eager, want))


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.layer_norm(x.cpu())
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x.half(), out_dtype=torch.float32),
                lambda: ops.layer_norm(x.half(), out_dtype=torch.bfloat16), lambda: ops.layer_norm_backward(x, x.half())):
        with pytest.raises(TypeError):
            bad()
    w = torch.ones(64, device="cuda")
    for bad in (lambda: ops.layer_norm(x, w[:32]), lambda: ops.layer_norm(x, w, w.cpu()), lambda: ops.layer_norm(x, eps=-1.0),
                lambda: ops.layer_norm_backward(x[:2], x), lambda: ops.layer_norm(x[:, :0])):
        with pytest.raises(ValueError):
            bad()
    # in place is refused where rows are read again
    big = torch.randn(2, 9000, device="cuda")
    a = _capi.LayerNormArgs()
    a.rows, a.dim, a.x_dtype, a.y_dtype, a.eps = 2, 9000, _capi.SUBQ_FP32, _capi.SUBQ_FP32, 1e-5
    a.x = a.dy = a.dx = big.data_ptr()
    a.x_stride = a.dy_stride = a.dx_stride = 9000
    with pytest.raises(ValueError, match="dx must not be"):
        _capi.layer_norm_bwd(a)


@pytest.mark.parametrize("x,y", [("fp32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("D", [72, 96, 384, 768, 896, 1280, 1536, 1544, 2048, 2056, 3080, 6144,
                               17, 129, 255, 257, 511, 515, 767, 1023, 1027, 2047, 2051, 4095, 6001])
def test_every_number_of_threads_a_row(D, x, y):
    """Widths on both sides of each step in the threads that hold a row, with rows enough for every CTA to loop."""
    shape = (min(40007, 6000000 // D), D)
    v, w, b, dy = make(shape, x, y, seed=D)
    ry, rdx, rdw, rdb = reference(v, w, b, 1e-5, dy)
    assert rel(ops.layer_norm(v, w, b, 1e-5, out_dtype=T[y]), ry) < tol(T[y])
    dx, dw, db = ops.layer_norm_backward(dy, v, w, 1e-5)
    assert rel(dx, rdx) < tol(T[x]) and rel(dw, rdw) < 3e-6 and rel(db, rdb) < 3e-6
