"""Outputs of the gated delta rule and of layer norm that share memory with an input, another output or themselves are
refused before anything is launched, and interleaved buffers that share none are not. (No call here has the workspace that
it needs, so what is not refused stops there.)"""
import ctypes
import random

import pytest

from subq_audio import _capi
from test_delta_capi import _bwd, _code, _fwd, _ln

APART, SHARED, ROWS = _capi.SUBQ_ERR_WORKSPACE, _capi.SUBQ_ERR_ALIAS, _capi.SUBQ_ERR_INVALID_ARGUMENT


def place(t, at, sb, sh, sn):
    t.data, t.stride_b, t.stride_h, t.stride_n = at, sb, sh, sn


def test_an_output_at_an_offset_into_another_tensor():
    for name in ("q", "k", "v"):
        for off in (2, 64 * 2, 50 * 64 * 2, 2 * 4 * 100 * 64 * 2 - 2, -2, -(2 * 4 * 100 * 64 * 2 - 2)):
            a = _fwd()
            a.o.data = getattr(a, name).data + off
            assert _code("subq_delta_fwd", a) == SHARED
            message = _capi.load().subq_last_error()
            assert b"o shares memory with" in message and name.encode() in message
        for off in (2 * 4 * 100 * 64 * 2, -2 * 4 * 100 * 64 * 2):
            a = _fwd()
            a.o.data = getattr(a, name).data + off
            assert _code("subq_delta_fwd", a) == APART
    for out in ("dq", "dk", "dv"):
        for name in ("q", "k", "v", "dout", "dq", "dk", "dv"):
            if name != out:
                a = _bwd()
                getattr(a, out).data = getattr(a, name).data + 130
                assert _code("subq_delta_bwd", a) == SHARED, (out, name)


def test_interleaved_views_of_one_buffer():
    B, H, N, d = 2, 4, 100, 64
    for heads_first in (False, True):  # [B, N, H, 4 d] and [B, N, 4, H, d]
        a = _fwd(B, H, N, d, d)
        for i, name in enumerate(("q", "k", "v", "o")):
            at, sh = (i * d * 2, 4 * d) if heads_first else (i * H * d * 2, d)
            place(getattr(a, name), 0x100000 + at, N * 4 * H * d, sh, 4 * H * d)
        assert _code("subq_delta_fwd", a) == APART
        a.o.data -= 2  # one element into v
        assert _code("subq_delta_fwd", a) == SHARED


def test_states_gates_and_masks():
    state = 2 * 4 * 64 * 64 * 4
    a = _fwd()
    a.state_in = a.state_out = 0x8000000
    assert _code("subq_delta_fwd", a) == APART  # in place
    for off in (4, state - 4, -4, 4 - state):
        a.state_out = a.state_in + off
        assert _code("subq_delta_fwd", a) == SHARED
    a.state_out = a.state_in + state
    assert _code("subq_delta_fwd", a) == APART
    a.state_out = a.o.data + 64
    assert _code("subq_delta_fwd", a) == SHARED
    a = _fwd()
    a.desc.beta.data, a.desc.beta.stride_b, a.desc.beta.stride_h, a.desc.beta.stride_n = a.o.data, 400, 100, 1
    assert _code("subq_delta_fwd", a) == SHARED
    a = _fwd()
    a.desc.mask, a.desc.mask_stride_b = a.o.data + 11, 100
    assert _code("subq_delta_fwd", a) == SHARED
    b = _bwd()
    b.state_in, b.dstate_out, b.dstate_in, b.dlog_gamma = 0x8000000, 0x9000000, 0x9000000, 0x11000000
    assert _code("subq_delta_bwd", b) == APART
    for field, value in (("dstate_in", 0x9000000 + state - 4), ("dstate_in", 0x8000000), ("dbeta", 0x11000000 + 2 * 4 * 100 * 4 - 4),
                         ("dlog_gamma", b.dq.data + 8), ("dbeta", b.dout.data)):
        c = _bwd()
        c.state_in, c.dstate_out, c.dstate_in, c.dlog_gamma = 0x8000000, 0x9000000, 0x9000000, 0x11000000
        setattr(c, field, value)
        assert _code("subq_delta_bwd", c) == SHARED, field


def test_rows_of_an_output_that_overlap():
    for strides in ((0, 100 * 64, 64), (4 * 100 * 64, 0, 64), (4 * 100 * 64, 100 * 64, 0), (4 * 100 * 64, 100 * 64, 63), (4 * 100 * 64 - 1, 100 * 64, 64),
                    (4 * 64, 64, 4 * 64)):
        a = _fwd()
        place(a.o, a.o.data, *strides)
        assert _code("subq_delta_fwd", a) == (APART if strides[2] == 64 and strides[:2] == (4 * 100 * 64, 100 * 64) else ROWS), strides
        for name in ("dq", "dk", "dv"):
            b = _bwd()
            place(getattr(b, name), getattr(b, name).data, *strides)
            assert _code("subq_delta_bwd", b) == ROWS, (strides, name)
    a = _fwd(B=1)
    place(a.o, a.o.data, 0, 64, 4 * 64)  # a stride of a single batch row says nothing
    assert _code("subq_delta_fwd", a) == APART
    a.q.stride_h = a.k.stride_n = 0  # inputs may be broadcast
    assert _code("subq_delta_fwd", a) == APART


def test_against_every_byte():
    """Random small strides, offsets and sizes: refused exactly where two rows share a byte."""
    rng = random.Random(5)
    seen = {APART: 0, SHARED: 0, ROWS: 0}
    for _ in range(3000):
        B, H, N, d, e = rng.randint(1, 3), rng.choice([1, 2, 4]), rng.randint(1, 5), rng.randint(1, 6), rng.randint(1, 6)
        a = _fwd(B, H, N, d, e)
        a.desc.path = 3  # (chunks: a workspace is needed)
        nested = rng.random() < 0.7
        rows = {}
        for name, width, heads in (("q", d, rng.choice([h for h in (1, 2, 4) if H % h == 0])), ("o", e, H)):
            t = getattr(a, name)
            at = 0x1000000 + 2 * rng.randint(0, 60)
            if nested:
                order, step, st = rng.sample(range(3), 3), width + rng.randint(0, 8), [0, 0, 0]
                for i in order:
                    st[i] = step
                    step *= (B, heads, N)[i]
            else:
                st = [rng.randint(0, 40) for _ in range(3)]
            place(t, at, *st)
            if name == "q":
                a.desc.q_heads = heads
            rows[name] = [range(p, p + 2 * width) for b in range(B) for h in range(heads) for n in range(N)
                          for p in [at + 2 * (b * st[0] + h * st[1] + n * st[2])]]
        own, other = [x for r in rows["o"] for x in r], {x for r in rows["q"] for x in r}
        want = ROWS if len(set(own)) < len(own) else SHARED if other & set(own) else APART
        if a.q.data == a.o.data and want == ROWS:
            want = SHARED  # (equal addresses are refused first)
        assert _code("subq_delta_fwd", a) == want
        seen[want] += 1
    assert min(seen.values()) > 200


def test_layer_norm():
    row = 64 * 4
    for field, base in (("dx", "x"), ("dx", "dy")):
        for off in (4, row, 9 * row, -4):
            a = _ln(y=_capi.SUBQ_FP32)
            a.dweight = 0x5000000
            setattr(a, field, getattr(a, base) + off)
            assert _code("subq_layer_norm_bwd", a) == SHARED
    for off in (4, row, 9 * row, -4):
        a = _ln(y=_capi.SUBQ_FP32)
        a.y = a.x + off
        assert _code("subq_layer_norm_fwd", a) == SHARED
    a = _ln(y=_capi.SUBQ_FP32)
    a.weight = a.y + row
    assert _code("subq_layer_norm_fwd", a) == SHARED
    for fields in (dict(dbias=0x5000000 + row - 4), dict(dbias=0x1000000), dict(weight=0x5000004), dict(dx=0x5000000 - 10 * row + 4)):
        a = _ln(y=_capi.SUBQ_FP32)
        a.dweight = 0x5000000
        for name, value in fields.items():
            setattr(a, name, value)
        assert _code("subq_layer_norm_bwd", a) == SHARED, fields
    # in place, and the columns between another tensor's
    for base in ("x", "dy"):
        a = _ln(y=_capi.SUBQ_FP32)
        a.dweight, a.dx = 0x5000000, getattr(a, base)
        assert _code("subq_layer_norm_bwd", a) == APART
    a = _ln(y=_capi.SUBQ_FP32)
    a.dweight, a.x_stride, a.dx_stride, a.dx = 0x5000000, 128, 128, a.x + row
    assert _code("subq_layer_norm_bwd", a) == APART


@pytest.mark.parametrize("make,call,name", [(_fwd, "subq_delta_fwd", "o"), (_bwd, "subq_delta_bwd", "dq")])
def test_strides_near_64_bits_end(make, call, name):
    a = make()
    place(getattr(a, name), getattr(a, name).data, 1 << 60, 1 << 50, 64)
    assert _code(call, a) == APART
    assert ctypes.sizeof(ctypes.c_void_p) == 8
