"""The C ABI of the selective state space block's operators: struct layouts, sizes, and refusals before anything is launched."""
import ctypes
import os
import subprocess

import pytest
import torch

from subq_audio import _capi, ops

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, ALIAS, NO, WS = _capi.SUBQ_ERR_INVALID_ARGUMENT, _capi.SUBQ_ERR_ALIAS, _capi.SUBQ_ERR_UNSUPPORTED, _capi.SUBQ_ERR_WORKSPACE


def test_struct_layout_matches_header(tmp_path):
    sizes = [("subq_tensor3", _capi.Tensor3), ("subq_selective_desc", _capi.SelectiveDesc), ("subq_selective_fwd_args", _capi.SelectiveFwdArgs),
             ("subq_selective_bwd_args", _capi.SelectiveBwdArgs), ("subq_causal_conv_args", _capi.CausalConvArgs),
             ("subq_rms_norm_args", _capi.RmsNormArgs), ("subq_scaled_matmul_args", _capi.ScaledMatmulArgs)]
    fields = [(c, p, f) for c, p in sizes for f, *_ in p._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "kernels.hpp"\nint main(void){'
                   + "".join(f'printf("%zu\\n", sizeof({c}));' for c, _ in sizes)
                   + "".join(f'printf("%zu\\n", offsetof({c}, {f}));' for c, _, f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-x", "c", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [ctypes.sizeof(p) for _, p in sizes] + [getattr(p, f).offset for _, p, f in fields]


def _code(call, a):
    return getattr(_capi.load(), call)(ctypes.byref(a))


def _scan(cls, names, B=2, L=100, D=64, N=16, G=2):
    a = cls()
    d = a.desc
    d.batch, d.seq_len, d.channels, d.states, d.groups, d.dtype, d.softplus = B, L, D, N, G, _capi.SUBQ_BF16, 1
    d.A, d.D, d.dt_bias = 0x9000000, 0x9100000, 0x9200000
    for i, name in enumerate(names):
        width = G * N if name in ("B", "C", "dB", "dC") else D
        t = getattr(a, name)
        t.data, t.stride_b, t.stride_l, t.stride_g = 0x100000 * (i + 1), L * width, width, N
    return a


def _fwd(**k):
    return _scan(_capi.SelectiveFwdArgs, ("u", "dt", "z", "B", "C", "out"), **k)


def _bwd(**k):
    a = _scan(_capi.SelectiveBwdArgs, ("u", "dt", "z", "B", "C", "dout", "du", "ddt", "dz", "dB", "dC"), **k)
    a.dA, a.dD, a.ddt_bias = 0xA000000, 0xA100000, 0xA200000
    return a


@pytest.mark.parametrize("field,value,code", [
    ("batch", -1, BAD), ("batch", 65536, BAD), ("seq_len", (1 << 30) + 1, BAD), ("channels", -2, BAD), ("channels", (1 << 24) + 2, BAD), ("channels", 63, BAD),
    ("states", 0, BAD), ("states", 129, NO), ("groups", 0, BAD), ("groups", 3, BAD), ("dtype", 3, BAD), ("dtype", 4, BAD), ("softplus", 2, BAD),
    ("A", None, BAD), ("A", 2, BAD), ("D", 0x9100002, BAD), ("dt_bias", 1, BAD),
])
def test_scan_descriptions(field, value, code):
    for call, a in (("subq_selective_scan_fwd", _fwd()), ("subq_selective_scan_bwd", _bwd())):
        setattr(a.desc, field, value)
        assert _code(call, a) == code
    assert _capi.load().subq_selective_scan_fwd(None) == BAD and _capi.load().subq_selective_scan_bwd(None) == BAD


def test_scan_tensors():
    for name in ("u", "dt", "B", "C", "out"):
        a = _fwd()
        getattr(a, name).data = None
        assert _code("subq_selective_scan_fwd", a) == BAD
        a = _fwd()
        getattr(a, name).data = 0x100001
        assert _code("subq_selective_scan_fwd", a) == BAD
        a = _fwd()
        getattr(a, name).stride_l = -1
        assert _code("subq_selective_scan_fwd", a) == BAD
    for name in ("u", "dt", "z", "B", "C"):
        a = _fwd()
        a.out.data = getattr(a, name).data + 2
        assert _code("subq_selective_scan_fwd", a) == ALIAS
        a = _bwd()
        a.dz.data = getattr(a, name).data
        assert _code("subq_selective_scan_bwd", a) == ALIAS
    a = _fwd()
    a.out.stride_l = 63  # rows that overlap
    assert _code("subq_selective_scan_fwd", a) == BAD
    a = _bwd()
    a.du.data = a.ddt.data
    assert _code("subq_selective_scan_bwd", a) == ALIAS
    a = _bwd()
    a.dA = a.ddt_bias
    assert _code("subq_selective_scan_bwd", a) == ALIAS
    a = _bwd()
    a.dA = None
    assert _code("subq_selective_scan_bwd", a) == BAD
    a = _fwd()
    a.mask, a.desc.mask = None, 0x5000000
    a.desc.mask_stride_b = -1
    assert _code("subq_selective_scan_fwd", a) == BAD
    a = _fwd()
    a.handover = 0xB000001
    assert _code("subq_selective_scan_fwd", a) == WS


def test_scan_workspaces():
    assert _capi.selective_scan_fwd_workspace_bytes(_fwd(B=64, D=1536, L=512, G=1)) == 0  # enough channels
    a = _fwd(B=1, D=64, L=4096, G=1)
    assert _capi.selective_scan_fwd_workspace_bytes(a) > 0
    assert _code("subq_selective_scan_fwd", a) == WS
    a.workspace, a.workspace_bytes = 0xC000001, 1 << 30
    assert _code("subq_selective_scan_fwd", a) == WS
    b = _bwd()
    with_states = _capi.selective_scan_bwd_workspace_bytes(b)
    assert _code("subq_selective_scan_bwd", b) == WS
    b.handover = 0xB000000
    handed = _capi.selective_scan_bwd_workspace_bytes(b)
    kept = _capi.selective_scan_handover_bytes(b.desc)
    assert kept == 2 * 13 * 64 * 16 * 4 and with_states - handed == kept  # 13 states of 100 tokens
    empty = _fwd(B=0)
    assert _code("subq_selective_scan_fwd", empty) == _capi.SUBQ_OK and _capi.load().subq_last_launches() == 0


def _conv(bwd=False, B=2, L=50, D=64, W=4):
    a = _capi.CausalConvArgs()
    a.batch, a.seq_len, a.channels, a.width, a.dtype, a.silu = B, L, D, W, _capi.SUBQ_FP16, 1
    for i, name in enumerate(("x", "y", "dy", "dx")):
        t = getattr(a, name)
        t.data, t.stride_b, t.stride_l = 0x100000 * (i + 1), L * D, D
    a.weight, a.bias = 0x9000000, 0x9100000
    if bwd:
        a.dweight, a.dbias = 0xA000000, 0xA100000
    return a


@pytest.mark.parametrize("field,value,code", [
    ("batch", -1, BAD), ("batch", 70000, BAD), ("seq_len", -1, BAD), ("channels", -1, BAD), ("width", 1, NO), ("width", 5, NO), ("dtype", 3, BAD), ("silu", 2, BAD),
    ("weight", None, BAD), ("weight", 1, BAD), ("bias", 2, BAD), ("state_in", 1, BAD),
])
def test_conv_descriptions(field, value, code):
    for call, a in (("subq_causal_conv_fwd", _conv()), ("subq_causal_conv_bwd", _conv(True))):
        setattr(a, field, value)
        assert _code(call, a) == code


def test_conv_memory():
    a = _conv()
    a.y.data = a.x.data
    assert _code("subq_causal_conv_fwd", a) == ALIAS
    a = _conv()
    a.state_in, a.state_out = 0x8000000, 0x8000002  # the same window, shifted by an element
    assert _code("subq_causal_conv_fwd", a) == ALIAS
    a = _conv(True)
    a.dx.data = a.dy.data
    assert _code("subq_causal_conv_bwd", a) == ALIAS
    a = _conv(True)
    assert _capi.causal_conv_bwd_workspace_bytes(a) > 0 and _code("subq_causal_conv_bwd", a) == WS
    a = _conv(True)
    a.dstate_out = a.dstate_in = 0x8000000
    assert _code("subq_causal_conv_bwd", a) == ALIAS
    a = _conv(True)
    a.dweight = None
    assert _code("subq_causal_conv_bwd", a) == BAD
    assert _code("subq_causal_conv_fwd", _conv(B=0)) == _capi.SUBQ_OK


def _norm(rows=10, dim=256):
    a = _capi.RmsNormArgs()
    a.rows, a.dim, a.eps, a.norm = rows, dim, 1e-5, 1
    a.x_dtype = a.r_dtype = a.y_dtype = _capi.SUBQ_BF16
    for i, name in enumerate(("x", "residual", "r", "y", "dy", "dr_next", "dx", "dres")):
        setattr(a, name, 0x100000 * (i + 1))
        setattr(a, name + "_stride", dim)
    a.weight, a.scale, a.scale_stride = 0x9000000, 0x9100000, 2
    return a


@pytest.mark.parametrize("field,value,code", [
    ("rows", -1, BAD), ("dim", 0, BAD), ("dim", 16385, NO), ("x_dtype", 3, BAD), ("r_dtype", _capi.SUBQ_FP16, NO), ("eps", -1.0, BAD), ("eps", float("nan"), BAD),
    ("norm", 2, BAD), ("r_stride", -1, BAD), ("weight", 2, BAD),
])
def test_norm_descriptions(field, value, code):
    for call in ("subq_rms_norm_fwd", "subq_rms_norm_bwd"):
        a = _norm()
        setattr(a, field, value)
        assert _code(call, a) == code


def test_norm_memory():
    for field, value, code in (("y_dtype", _capi.SUBQ_FP32, NO), ("y_dtype", 3, NO), ("x", None, BAD), ("y", None, BAD), ("y", 0x100000, ALIAS), ("y", 0x200000, ALIAS),
                               ("r", 0x100002, ALIAS), ("y_stride", 255, BAD), ("r", 0x400000, ALIAS)):
        a = _norm()
        setattr(a, field, value)
        assert _code("subq_rms_norm_fwd", a) == code, (field, value)
    a = _norm()
    a.y_dtype, a.scale = _capi.SUBQ_E4M3, None
    assert _code("subq_rms_norm_fwd", a) == BAD
    a = _norm()
    a.y_dtype, a.scale_stride = _capi.SUBQ_E4M3, 1
    assert _code("subq_rms_norm_fwd", a) == BAD
    for field, value, code in (("dy", None, BAD), ("r", None, BAD), ("dx", 0x300000, ALIAS), ("dres", 0x500000, ALIAS), ("dx", 0x800000, ALIAS), ("dres_stride", 9, BAD)):
        a = _norm()
        setattr(a, field, value)
        assert _code("subq_rms_norm_bwd", a) == code, (field, value)
    a = _norm()
    a.dweight = 0xA000000
    assert _capi.rms_norm_bwd_workspace_bytes(a) > 0 and _code("subq_rms_norm_bwd", a) == WS
    assert _code("subq_rms_norm_fwd", _norm(rows=0)) == _capi.SUBQ_OK


def _mm(M=100, N=200, K=300):
    a = _capi.ScaledMatmulArgs()
    a.M, a.N, a.K, a.out_dtype = M, N, K, _capi.SUBQ_BF16
    a.a, a.a_stride, a.b, a.b_stride = 0x100000, 304, 0x200000, 304
    a.a_scale, a.a_scale_stride, a.b_scale, a.b_scale_stride = 0x300000, 3, 0x400000, 3
    a.out, a.out_stride = 0x500000, N
    return a


@pytest.mark.parametrize("field,value,code", [
    ("M", -1, BAD), ("N", -1, BAD), ("K", -1, BAD), ("M", (1 << 30) + 1, BAD), ("N", 1 << 25, BAD), ("K", 1 << 25, BAD), ("out_dtype", 3, BAD), ("out_dtype", 4, BAD),
    ("a", None, BAD), ("a", 0x100008, BAD), ("a_stride", 300, BAD), ("a_stride", 288, BAD), ("b_stride", 1 << 41, BAD), ("b", 0x200001, BAD), ("a_scale", None, BAD),
    ("b_scale", 0x400002, BAD), ("a_scale_stride", -3, BAD), ("out", None, BAD), ("out", 0x500001, BAD), ("out_stride", 199, BAD), ("out", 0x100000, ALIAS),
    ("out", 0x300000, ALIAS), ("bias", 2, BAD),
])
def test_product(field, value, code):
    a = _mm()
    setattr(a, field, value)
    assert _code("subq_scaled_matmul", a) == code
    assert _capi.load().subq_scaled_matmul(None) == BAD


def test_product_of_nothing():
    assert _code("subq_scaled_matmul", _mm(M=0)) == _capi.SUBQ_OK and _code("subq_scaled_matmul", _mm(N=0)) == _capi.SUBQ_OK


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8, 16)
    b = torch.zeros(2, 8, 4)
    for call in (lambda: ops.causal_conv_forward(x, torch.zeros(16, 4)), lambda: ops.selective_scan_forward(x, x, torch.zeros(16, 4), b, b),
                 lambda: ops.rms_norm(x), lambda: ops.rms_norm_fp8(x), lambda: ops.quantize_fp8(x),
                 lambda: ops.scaled_matmul(x.to(torch.float8_e4m3fn), x, x[0].to(torch.float8_e4m3fn), x)):
        with pytest.raises(RuntimeError):
            call()
