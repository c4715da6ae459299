"""The C ABI of the gated delta rule and of layer norm: struct layouts, sizes, and refusals before anything is launched."""
import ctypes
import os
import subprocess

import pytest

from subq_audio import _capi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header(tmp_path):
    sizes = [("subq_gate", _capi.Gate), ("subq_delta_desc", _capi.DeltaDesc), ("subq_delta_fwd_args", _capi.DeltaFwdArgs),
             ("subq_delta_bwd_args", _capi.DeltaBwdArgs), ("subq_layer_norm_args", _capi.LayerNormArgs)]
    fields = [(c, p, f) for c, p in sizes for f, *_ in p._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "kernels.hpp"\nint main(void){'
                   + "".join(f'printf("%zu\\n", sizeof({c}));' for c, _ in sizes)
                   + "".join(f'printf("%zu\\n", offsetof({c}, {f}));' for c, _, f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-x", "c", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [ctypes.sizeof(p) for _, p in sizes] + [getattr(p, f).offset for _, p, f in fields]


def _fill(a, names, B, H, N, d, e):
    a.desc.batch, a.desc.heads, a.desc.seq_len, a.desc.head_dim, a.desc.value_dim = B, H, N, d, e
    a.desc.dtype, a.desc.scale = _capi.SUBQ_BF16, 0.125
    for i, (name, width) in enumerate(names):
        t = getattr(a, name)
        t.data = 0x100000 * (i + 1)
        t.stride_b, t.stride_h, t.stride_n = H * N * width, N * width, width
    return a


def _fwd(B=2, H=4, N=100, d=64, e=64):
    return _fill(_capi.DeltaFwdArgs(), (("q", d), ("k", d), ("v", e), ("o", e)), B, H, N, d, e)


def _bwd(B=2, H=4, N=100, d=64, e=64):
    a = _fill(_capi.DeltaBwdArgs(), (("q", d), ("k", d), ("v", e), ("dout", e), ("dq", d), ("dk", d), ("dv", e)), B, H, N, d, e)
    a.dbeta = 0x10000000
    return a


def _code(call, a):
    return getattr(_capi.load(), call)(ctypes.byref(a))


@pytest.mark.parametrize("field,value,code", [
    ("batch", -1, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("batch", 65536, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("seq_len", (1 << 30) + 1, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("head_dim", 0, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("head_dim", 257, _capi.SUBQ_ERR_UNSUPPORTED),
    ("value_dim", 512, _capi.SUBQ_ERR_UNSUPPORTED),
    ("dtype", 3, _capi.SUBQ_ERR_INVALID_ARGUMENT),  # float64
    ("dtype", 9, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("path", 2, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("q_heads", 3, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("k_heads", 8, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("v_heads", -1, _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("scale", float("nan"), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    ("scale", float("inf"), _capi.SUBQ_ERR_INVALID_ARGUMENT),
])
@pytest.mark.parametrize("call,make", [("subq_delta_fwd", _fwd), ("subq_delta_bwd", _bwd)])
def test_delta_rejects_bad_descriptions(call, make, field, value, code):
    a = make()
    setattr(a.desc, field, value)
    assert _code(call, a) == code


@pytest.mark.parametrize("call,make,names", [
    ("subq_delta_fwd", _fwd, ("q", "k", "v", "o")),
    ("subq_delta_bwd", _bwd, ("q", "k", "v", "dout", "dq", "dk", "dv")),
])
def test_delta_rejects_bad_tensors(call, make, names):
    for name in names:
        for field, value in (("data", None), ("data", 0x1001), ("stride_h", -64)):
            a = make()
            setattr(getattr(a, name), field, value)
            assert _code(call, a) == _capi.SUBQ_ERR_INVALID_ARGUMENT, (name, field)
            assert name.encode() in _capi.load().subq_last_error()
    for gate in ("beta", "log_gamma"):
        a = make()
        getattr(a.desc, gate).data = 0x1002
        assert _code(call, a) == _capi.SUBQ_ERR_INVALID_ARGUMENT
        getattr(a.desc, gate).data, getattr(a.desc, gate).stride_n = 0x1000, -1
        assert _code(call, a) == _capi.SUBQ_ERR_INVALID_ARGUMENT
    a = make()
    a.desc.mask, a.desc.mask_stride_b = 0x1000, -1
    assert _code(call, a) == _capi.SUBQ_ERR_INVALID_ARGUMENT


def test_delta_rejects_aliases():
    for name in ("q", "k", "v"):
        a = _fwd()
        a.o.data = getattr(a, name).data
        assert _code("subq_delta_fwd", a) == _capi.SUBQ_ERR_ALIAS
    for out in ("dq", "dk", "dv"):
        for name in ("q", "k", "v", "dout", "dq", "dk", "dv"):
            if name != out:
                a = _bwd()
                getattr(a, out).data = getattr(a, name).data
                assert _code("subq_delta_bwd", a) == _capi.SUBQ_ERR_ALIAS, (out, name)
    a = _bwd()
    a.dbeta = None
    assert _code("subq_delta_bwd", a) == _capi.SUBQ_ERR_INVALID_ARGUMENT


def test_delta_paths_and_head_sizes():
    a = _fwd(d=160)
    a.desc.path = 3
    assert _code("subq_delta_fwd", a) == _capi.SUBQ_ERR_UNSUPPORTED  # chunks need d <= 128
    a.desc.path = 1
    a.handover = 0x1000000
    assert _code("subq_delta_fwd", a) == _capi.SUBQ_ERR_UNSUPPORTED  # the recurrent kernel fills none
    assert _capi.delta_handover_bytes(a.desc) == 0
    assert _code("subq_delta_bwd", _bwd(d=160)) == _capi.SUBQ_ERR_UNSUPPORTED
    a = _bwd()
    a.desc.path = 1
    assert _code("subq_delta_bwd", a) == _capi.SUBQ_ERR_UNSUPPORTED


def test_delta_workspaces():
    assert _capi.delta_fwd_workspace_bytes(_fwd(N=1)) == 0  # recurrent
    a = _fwd()
    need = _capi.delta_fwd_workspace_bytes(a)
    assert need > 0
    for ws, have in ((None, need), (0x1000000, need - 1), (0x1000010, need)):
        a.workspace, a.workspace_bytes = ws, have
        assert _code("subq_delta_fwd", a) == _capi.SUBQ_ERR_WORKSPACE
    a.workspace, a.workspace_bytes, a.handover = 0x1000000, need, 0x1000010
    assert _code("subq_delta_fwd", a) == _capi.SUBQ_ERR_WORKSPACE
    b = _bwd()
    full = _capi.delta_bwd_workspace_bytes(b)
    b.handover = 0x1000000
    part = _capi.delta_bwd_workspace_bytes(b)
    assert 0 < part < full and full - part >= _capi.delta_handover_bytes(b.desc)
    b.workspace, b.workspace_bytes = 0x2000000, part - 1
    assert _code("subq_delta_bwd", b) == _capi.SUBQ_ERR_WORKSPACE
    # gradients per state head of shared heads
    b.desc.k_heads = 2
    assert _capi.delta_bwd_workspace_bytes(b) == part + 2 * 4 * 100 * 64 * 4
    # a state updated in place by several segments needs a copy of it
    a = _fwd(B=1, H=4, N=4096)
    a.state_in, a.state_out = 0x4000000, 0x5000000
    apart = _capi.delta_fwd_workspace_bytes(a)
    a.state_out = a.state_in
    assert _capi.delta_fwd_workspace_bytes(a) == apart + 4 * 64 * 64 * 4
    # many sequences are not cut up
    a = _fwd(B=8, H=32, N=4096)
    a.state_in = a.state_out = 0x4000000
    same = _capi.delta_fwd_workspace_bytes(a)
    a.state_out = None
    assert _capi.delta_fwd_workspace_bytes(a) == same


def test_delta_sizes_pass_32_bits():
    a = _fwd(B=16, H=64, N=1 << 20)
    assert _capi.delta_handover_bytes(a.desc) > 1 << 32
    a = _fwd(B=4096, H=4096, N=1 << 14)
    assert _code("subq_delta_fwd", a) == _capi.SUBQ_ERR_UNSUPPORTED  # more CTAs than a grid has
    assert _capi.delta_fwd_workspace_bytes(a) == 0 and _capi.delta_handover_bytes(a.desc) == 0


@pytest.mark.parametrize("B,H,N", [(0, 4, 100), (2, 0, 100), (2, 4, 0)])
def test_delta_without_tokens_launches_nothing(B, H, N):
    for call, make in (("subq_delta_fwd", _fwd), ("subq_delta_bwd", _bwd)):
        a = make(B, H, N)
        for name in ("q", "k", "v"):
            getattr(a, name).data = None
        assert _code(call, a) == _capi.SUBQ_OK
        assert _capi.load().subq_last_launches() == 0


def test_null_argument_blocks():
    lib = _capi.load()
    for call in ("subq_delta_fwd", "subq_delta_bwd", "subq_layer_norm_fwd", "subq_layer_norm_bwd"):
        assert getattr(lib, call)(None) == _capi.SUBQ_ERR_INVALID_ARGUMENT
    for call in ("subq_delta_fwd_workspace_bytes", "subq_delta_bwd_workspace_bytes", "subq_delta_handover_bytes",
                 "subq_layer_norm_bwd_workspace_bytes"):
        assert getattr(lib, call)(None) == 0


def _ln(rows=10, dim=64, x=_capi.SUBQ_FP32, y=_capi.SUBQ_BF16):
    a = _capi.LayerNormArgs()
    a.rows, a.dim, a.x_dtype, a.y_dtype, a.eps = rows, dim, x, y, 1e-5
    a.x, a.y, a.dy, a.dx = 0x1000000, 0x2000000, 0x3000000, 0x4000000
    a.x_stride = a.y_stride = a.dy_stride = a.dx_stride = dim
    return a


LN_CALLS = pytest.mark.parametrize("call", ["subq_layer_norm_fwd", "subq_layer_norm_bwd"])


@LN_CALLS
@pytest.mark.parametrize("fields,code", [
    (dict(rows=-1), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(dim=0), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(dim=(1 << 24) + 1), _capi.SUBQ_ERR_UNSUPPORTED),
    (dict(x_dtype=3), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(x_dtype=_capi.SUBQ_BF16, y_dtype=_capi.SUBQ_FP32), _capi.SUBQ_ERR_UNSUPPORTED),
    (dict(x_dtype=_capi.SUBQ_FP16), _capi.SUBQ_ERR_UNSUPPORTED),
    (dict(eps=-1.0), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(eps=float("nan")), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(x=None), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(x=0x1002), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(x_stride=-64), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(y=None, dy=None), _capi.SUBQ_ERR_INVALID_ARGUMENT),
    (dict(y_stride=63, dx_stride=63), _capi.SUBQ_ERR_INVALID_ARGUMENT),  # rows of the output overlap
])
def test_layer_norm_rejects(call, fields, code):
    a = _ln()
    for name, value in fields.items():
        setattr(a, name, value)
    assert _code(call, a) == code


def test_layer_norm_in_place_needs_one_layout():
    a = _ln()
    a.y = a.x
    assert _code("subq_layer_norm_fwd", a) == _capi.SUBQ_ERR_ALIAS  # 16-bit rows over float32 ones
    a = _ln()
    a.dx = a.dy
    assert _code("subq_layer_norm_bwd", a) == _capi.SUBQ_ERR_ALIAS
    a = _ln()
    a.dx, a.dx_stride = a.x, 128
    assert _code("subq_layer_norm_bwd", a) == _capi.SUBQ_ERR_ALIAS
    a = _ln(dim=8193, y=_capi.SUBQ_FP32)
    a.dx = a.x
    assert _code("subq_layer_norm_bwd", a) == _capi.SUBQ_ERR_ALIAS  # long rows are read more than once


def test_layer_norm_workspace():
    a = _ln()
    assert _capi.layer_norm_bwd_workspace_bytes(a) == 0  # neither sum is wanted
    a.dweight = 0x5000000
    need = _capi.layer_norm_bwd_workspace_bytes(a)
    assert need >= 2 * 10 * 64 * 4
    for ws, have in ((None, need), (0x6000000, need - 1), (0x6000004, need)):
        a.workspace, a.workspace_bytes = ws, have
        assert _code("subq_layer_norm_bwd", a) == _capi.SUBQ_ERR_WORKSPACE
    a = _ln(rows=0)
    a.x = a.y = None
    assert _code("subq_layer_norm_fwd", a) == _capi.SUBQ_OK


def test_state_gradient_in_place_is_not_cut_into_segments():
    b = _bwd(B=1, H=4, N=4096)
    b.dstate_out, b.dstate_in = 0x20000000, 0x30000000
    cut = _capi.delta_bwd_workspace_bytes(b)
    b.dstate_in = b.dstate_out
    assert 0 < _capi.delta_bwd_workspace_bytes(b) < cut
