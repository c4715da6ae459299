"""The scan as torch operators: ``torch.ops.subq_audio.scan_fwd`` and
``torch.ops.subq_audio.scan_bwd`` (normalised form, the model path of
``SubQLinearAttention`` / ``chunkwise_flash_linear_attention``).

Registered with ``torch.library`` with fake (meta) kernels, so a model that
calls them can be traced by ``torch.compile`` / ``torch.export`` without a
graph break: the fake kernels give the outputs' shapes, dtypes and memory
order (the output follows q's memory order, as ``ops.scan_forward`` writes
it) and the size of the forward's handover buffer, which is a function of
the shapes only. The real kernels are the C-ABI calls of ``ops``.

    o, S, z, handover = torch.ops.subq_audio.scan_fwd(q, k, v, log_gamma, mask, S0, z0, reverse, want_state)
    dq, dk, dv, dlog_gamma = torch.ops.subq_audio.scan_bwd(q, k, v, dout, log_gamma, mask, S0, z0, o,
                                                           handover, reverse, need_dlog_gamma)

``log_gamma`` is None or float32 ([], [H] or [B, H, N]); ``mask`` None or a
uint8 / bool [B, N]; ``S0`` [B, H, d, e] and ``z0`` [B, H, d] float32 or
None. Outputs that a call does not produce (S, z without ``want_state``, the
handover off the tensor-core path, d log(gamma) without ``need_dlog_gamma``)
are empty tensors.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _capi, ops

Tensor = torch.Tensor
_FAKE_PTR = 1 << 16  # a 16-byte-aligned stand-in address: the size query reads no memory


def _handover_bytes(q: Tensor, k: Tensor, v: Tensor, log_gamma: Optional[Tensor], mask: Optional[Tensor],
                    reverse: bool) -> int:
    """Bytes of the forward's handover buffer for these shapes and strides
    (subq_segment_states_bytes; no tensor data is read)."""
    B, H, N, d = q.shape
    a = _capi.FwdArgs()
    desc = a.desc
    desc.batch, desc.heads, desc.seq_len, desc.head_dim, desc.value_dim = B, H, N, d, v.shape[-1]
    desc.kv_heads = v.shape[1] if v.shape[1] != H else 0
    desc.dtype = ops._DTYPES[q.dtype]
    desc.normalize = 1
    desc.scale = 1.0 / math.sqrt(d)
    desc.clamp_min = 1e-5
    desc.path = _capi.SUBQ_PATH_AUTO
    desc.reverse = 1 if reverse else 0
    if log_gamma is not None:
        desc.decay_mode = _capi.SUBQ_DECAY_PER_TOKEN
        desc.log_gamma = _FAKE_PTR
    if mask is not None:
        desc.mask = _FAKE_PTR
        desc.mask_stride_b = N
    # (o is allocated in q's memory order; the size depends on its strides only
    # through their alignment, which q's share)
    for name, t in (("q", q), ("k", k), ("v", v), ("o", q)):
        t4 = getattr(a, name)
        t4.data = _FAKE_PTR
        t4.stride_b, t4.stride_h, t4.stride_n = t.stride(0), t.stride(1), t.stride(2)
    with torch.cuda.device(q.device):
        return _capi.segment_states_bytes(a)


def _empty_f32(ref: Tensor, shape) -> Tensor:
    return torch.empty(shape, dtype=torch.float32, device=ref.device)


@torch.library.custom_op("subq_audio::scan_fwd", mutates_args=(), device_types="cuda")
def scan_fwd(q: Tensor, k: Tensor, v: Tensor, log_gamma: Optional[Tensor], mask: Optional[Tensor],
             S0: Optional[Tensor], z0: Optional[Tensor], reverse: bool,
             want_state: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    seg = ops.SegmentStates()
    state = None if S0 is None else (S0, z0)
    o, st = ops.scan_forward(q, k, v, log_gamma=log_gamma, mask=mask, normalize=True, state=state,
                             return_state=want_state, reverse=reverse, segments=seg)
    S, z = st if want_state else (_empty_f32(q, (0,)), _empty_f32(q, (0,)))
    handover = seg.buf if seg.buf is not None else torch.empty(0, dtype=torch.uint8, device=q.device)
    return o, S, z, handover


@scan_fwd.register_fake
def _scan_fwd_fake(q, k, v, log_gamma, mask, S0, z0, reverse, want_state):
    B, H, N, d = q.shape
    e = v.shape[-1]
    o = ops._empty_in_order(q, (B, H, N, e), q.dtype)
    if want_state:
        S, z = _empty_f32(q, (B, H, d, e)), _empty_f32(q, (B, H, d))
    else:
        S, z = _empty_f32(q, (0,)), _empty_f32(q, (0,))
    nbytes = _handover_bytes(q, k, v, log_gamma, mask, reverse)
    return o, S, z, torch.empty(nbytes, dtype=torch.uint8, device=q.device)


@torch.library.custom_op("subq_audio::scan_bwd", mutates_args=(), device_types="cuda")
def scan_bwd(q: Tensor, k: Tensor, v: Tensor, dout: Tensor, log_gamma: Optional[Tensor], mask: Optional[Tensor],
             S0: Optional[Tensor], z0: Optional[Tensor], o: Tensor, handover: Tensor, reverse: bool,
             need_dlog_gamma: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    seg = None
    if handover.numel() > 0:
        seg = ops.SegmentStates()
        seg.buf = handover
    state = None if S0 is None else (S0, z0)
    dq, dk, dv, dlg = ops.scan_backward(q, k, v, dout, log_gamma=log_gamma, mask=mask, normalize=True, state=state,
                                        need_dlog_gamma=need_dlog_gamma, reverse=reverse, segments=seg,
                                        forward_out=o if seg is not None else None)
    if dlg is None:
        dlg = _empty_f32(q, (0,))
    return dq, dk, dv, dlg


@scan_bwd.register_fake
def _scan_bwd_fake(q, k, v, dout, log_gamma, mask, S0, z0, o, handover, reverse, need_dlog_gamma):
    B, H, N, _ = q.shape
    dq = ops._empty_in_order(q, tuple(q.shape), q.dtype)
    dk = ops._empty_in_order(k, tuple(k.shape), q.dtype)
    dv = ops._empty_in_order(v, tuple(v.shape), q.dtype)
    dlg = _empty_f32(q, (B, H, N) if need_dlog_gamma else (0,))
    return dq, dk, dv, dlg


# Per-head RMSNorm of the scan's output (the module epilogue):
#     y = torch.ops.subq_audio.head_rmsnorm_fwd(x, weight, eps)
#     dx, dweight = torch.ops.subq_audio.head_rmsnorm_bwd(dy, x, weight, eps)
# y is a [B, H, N, D] view of a [B, N, H, D] buffer; dweight is float32 [D]
# (empty without a weight).
@torch.library.custom_op("subq_audio::head_rmsnorm_fwd", mutates_args=(), device_types="cuda")
def head_rmsnorm_fwd(x: Tensor, weight: Optional[Tensor], eps: float) -> Tensor:
    return ops.head_rmsnorm(x, weight, eps)


@head_rmsnorm_fwd.register_fake
def _head_rmsnorm_fwd_fake(x, weight, eps):
    B, H, N, D = x.shape
    return x.new_empty((B, N, H, D)).transpose(1, 2)


@torch.library.custom_op("subq_audio::head_rmsnorm_bwd", mutates_args=(), device_types="cuda")
def head_rmsnorm_bwd(dy: Tensor, x: Tensor, weight: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor]:
    dx, dw = ops.head_rmsnorm_backward(dy, x, weight, eps, need_dweight=weight is not None)
    return dx, (dw if dw is not None else _empty_f32(x, (0,)))


@head_rmsnorm_bwd.register_fake
def _head_rmsnorm_bwd_fake(dy, x, weight, eps):
    dx = ops._empty_in_order(x, tuple(x.shape), x.dtype)
    return dx, _empty_f32(x, (x.shape[-1],) if weight is not None else (0,))


# The gated delta rule and its gradients:
#     o, S, handover = torch.ops.subq_audio.gated_delta_fwd(q, k, v, beta, log_gamma, mask, S0, scale, want_state, want_handover)
#     dq, dk, dv, dbeta, dlog_gamma, dS0 = torch.ops.subq_audio.gated_delta_bwd(q, k, v, beta, dout, log_gamma, mask, S0, dS,
#                                                                             scale, handover, need_dlog_gamma, need_dS0)
# beta and log_gamma are None or tensors [], [H] or [B, H, N]; dbeta and
# dlog_gamma come per token, [B, H, N] float32. What a call does not produce is
# an empty tensor; an empty handover lets the backward form it again.
def _delta_H(q: Tensor, k: Tensor, v: Tensor, beta: Optional[Tensor], log_gamma: Optional[Tensor]) -> int:
    return ops._delta_heads(q, k, v, beta, log_gamma)


def _delta_handover(q: Tensor, k: Tensor, v: Tensor, H: int) -> int:
    d = _capi.DeltaDesc()
    d.batch, d.heads, d.seq_len, d.head_dim, d.value_dim = q.shape[0], H, q.shape[2], q.shape[3], v.shape[3]
    d.q_heads, d.k_heads, d.v_heads, d.dtype, d.scale = q.shape[1], k.shape[1], v.shape[1], ops._DTYPES[q.dtype], 1.0
    return _capi.delta_handover_bytes(d)


@torch.library.custom_op("subq_audio::gated_delta_fwd", mutates_args=(), device_types="cuda")
def gated_delta_fwd(q: Tensor, k: Tensor, v: Tensor, beta: Optional[Tensor], log_gamma: Optional[Tensor],
                    mask: Optional[Tensor], S0: Optional[Tensor], scale: float, want_state: bool,
                    want_handover: bool) -> Tuple[Tensor, Tensor, Tensor]:
    ho = ops.DeltaHandover() if want_handover else None
    o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=log_gamma, mask=mask, scale=scale, state=S0,
                                   return_state=want_state, handover=ho)
    buf = ho.buf if ho is not None and ho.buf is not None else torch.empty(0, dtype=torch.uint8, device=q.device)
    return o, (S if want_state else _empty_f32(q, (0,))), buf


@gated_delta_fwd.register_fake
def _gated_delta_fwd_fake(q, k, v, beta, log_gamma, mask, S0, scale, want_state, want_handover):
    H = _delta_H(q, k, v, beta, log_gamma)
    B, _, N, d = q.shape
    o = ops._empty_in_order(q, (B, H, N, v.shape[-1]), q.dtype)
    S = _empty_f32(q, (B, H, d, v.shape[-1]) if want_state else (0,))
    return o, S, torch.empty(_delta_handover(q, k, v, H) if want_handover else 0, dtype=torch.uint8, device=q.device)


@torch.library.custom_op("subq_audio::gated_delta_bwd", mutates_args=(), device_types="cuda")
def gated_delta_bwd(q: Tensor, k: Tensor, v: Tensor, beta: Optional[Tensor], dout: Tensor, log_gamma: Optional[Tensor],
                    mask: Optional[Tensor], S0: Optional[Tensor], dS: Optional[Tensor], scale: float, handover: Tensor,
                    need_dlog_gamma: bool, need_dS0: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    ho = None
    if handover.numel() > 0:
        H = _delta_H(q, k, v, beta, log_gamma)
        ho = ops.DeltaHandover()
        ho.buf, ho.key = handover, (q.shape[0], H, q.shape[2], q.shape[3], v.shape[3], q.dtype, q.device)
    dq, dk, dv, dbeta, dlg, dS0 = ops.gated_delta_backward(q, k, v, beta, dout, log_gamma=log_gamma, mask=mask, scale=scale,
                                                           state=S0, dstate=dS, need_dlog_gamma=need_dlog_gamma,
                                                           need_dstate=need_dS0, handover=ho)
    return (dq, dk, dv, dbeta, dlg if dlg is not None else _empty_f32(q, (0,)),
            dS0 if dS0 is not None else _empty_f32(q, (0,)))


@gated_delta_bwd.register_fake
def _gated_delta_bwd_fake(q, k, v, beta, dout, log_gamma, mask, S0, dS, scale, handover, need_dlog_gamma, need_dS0):
    H = _delta_H(q, k, v, beta, log_gamma)
    B, _, N, d = q.shape
    return (ops._empty_in_order(q, tuple(q.shape), q.dtype), ops._empty_in_order(k, tuple(k.shape), q.dtype),
            ops._empty_in_order(v, tuple(v.shape), q.dtype), _empty_f32(q, (B, H, N)),
            _empty_f32(q, (B, H, N) if need_dlog_gamma else (0,)), _empty_f32(q, (B, H, d, v.shape[-1]) if need_dS0 else (0,)))


# Layer norm over the last dimension:
#     y = torch.ops.subq_audio.layer_norm_fwd(x, weight, bias, eps, out_dtype)
#     dx, dweight, dbias = torch.ops.subq_audio.layer_norm_bwd(dy, x, weight, eps, need_dweight, need_dbias)
@torch.library.custom_op("subq_audio::layer_norm_fwd", mutates_args=(), device_types="cuda")
def layer_norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                   out_dtype: Optional[torch.dtype]) -> Tensor:
    return ops.layer_norm(x, weight, bias, eps, out_dtype=out_dtype)


@layer_norm_fwd.register_fake
def _layer_norm_fwd_fake(x, weight, bias, eps, out_dtype):
    return torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)


@torch.library.custom_op("subq_audio::layer_norm_bwd", mutates_args=(), device_types="cuda")
def layer_norm_bwd(dy: Tensor, x: Tensor, weight: Optional[Tensor], eps: float, need_dweight: bool,
                   need_dbias: bool) -> Tuple[Tensor, Tensor, Tensor]:
    dx, dw, db = ops.layer_norm_backward(dy, x, weight, eps, need_dweight=need_dweight, need_dbias=need_dbias)
    return dx, (dw if dw is not None else _empty_f32(x, (0,))), (db if db is not None else _empty_f32(x, (0,)))


@layer_norm_bwd.register_fake
def _layer_norm_bwd_fake(dy, x, weight, eps, need_dweight, need_dbias):
    D = x.shape[-1]
    return (torch.empty(x.shape, dtype=x.dtype, device=x.device), _empty_f32(x, (D if need_dweight else 0,)),
            _empty_f32(x, (D if need_dbias else 0,)))


# The selective scan and its gradients:
#     out, S, handover = torch.ops.subq_audio.selective_scan_fwd(u, dt, A, B, C, D, z, dt_bias, mask, S0, dt_softplus, want_state,
#                                                                want_handover)
#     du, ddt, dA, dB, dC, dD, dz, ddt_bias, dS0 = torch.ops.subq_audio.selective_scan_bwd(u, dt, A, B, C, dout, D, z, dt_bias,
#                                                                mask, S0, dS, dt_softplus, handover, need_dS0)
# (shapes as in ops.selective_scan_forward). What a call does not produce is an empty tensor; an empty handover lets the
# backward form it again.
def _scan_groups(B: Tensor) -> int:
    return B.shape[2] if B.dim() == 4 else 1


def _scan_handover(u: Tensor, A: Tensor, B: Tensor) -> int:
    d = _capi.SelectiveDesc()
    d.batch, d.seq_len, d.channels, d.states, d.groups = *u.shape, A.shape[1], _scan_groups(B)
    d.dtype, d.A = ops._DTYPES[u.dtype], _FAKE_PTR
    return _capi.selective_scan_handover_bytes(d)


@torch.library.custom_op("subq_audio::selective_scan_fwd", mutates_args=(), device_types="cuda")
def selective_scan_fwd(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor], dt_bias: Optional[Tensor],
                       mask: Optional[Tensor], S0: Optional[Tensor], dt_softplus: bool, want_state: bool,
                       want_handover: bool) -> Tuple[Tensor, Tensor, Tensor]:
    ho = ops.ScanHandover() if want_handover else None
    y, S = ops.selective_scan_forward(u, dt, A, B, C, D=D, z=z, dt_bias=dt_bias, dt_softplus=dt_softplus, mask=mask, state=S0,
                                      return_state=want_state, handover=ho)
    return y, (S if want_state else _empty_f32(u, (0,))), (ho.buf if ho is not None else torch.empty(0, dtype=torch.uint8, device=u.device))


@selective_scan_fwd.register_fake
def _selective_scan_fwd_fake(u, dt, A, B, C, D, z, dt_bias, mask, S0, dt_softplus, want_state, want_handover):
    S = _empty_f32(u, (u.shape[0], u.shape[2], A.shape[1]) if want_state else (0,))
    return (torch.empty(u.shape, dtype=u.dtype, device=u.device), S,
            torch.empty(_scan_handover(u, A, B) if want_handover else 0, dtype=torch.uint8, device=u.device))


@torch.library.custom_op("subq_audio::selective_scan_bwd", mutates_args=(), device_types="cuda")
def selective_scan_bwd(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, dout: Tensor, D: Optional[Tensor], z: Optional[Tensor],
                       dt_bias: Optional[Tensor], mask: Optional[Tensor], S0: Optional[Tensor], dS: Optional[Tensor], dt_softplus: bool, handover: Tensor,
                       need_dS0: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    ho = None
    if handover.numel() > 0:
        ho = ops.ScanHandover()
        ho.buf, ho.key = handover, (tuple(u.shape), A.shape[1], _scan_groups(B), u.dtype, u.device)
    g = ops.selective_scan_backward(u, dt, A, B, C, dout, D=D, z=z, dt_bias=dt_bias, dt_softplus=dt_softplus, mask=mask, state=S0, dstate=dS,
                                    need_dstate=need_dS0, handover=ho)
    return tuple(x if x is not None else _empty_f32(u, (0,)) for x in g)


@selective_scan_bwd.register_fake
def _selective_scan_bwd_fake(u, dt, A, B, C, dout, D, z, dt_bias, mask, S0, dS, dt_softplus, handover, need_dS0):
    def like(t):
        return _empty_f32(u, (0,)) if t is None else torch.empty(t.shape, dtype=t.dtype, device=u.device)

    Dn = u.shape[2]
    return (like(u), like(dt), _empty_f32(u, A.shape), like(B), like(C), _empty_f32(u, (0 if D is None else Dn,)), like(z),
            _empty_f32(u, (0 if dt_bias is None else Dn,)), _empty_f32(u, (u.shape[0], Dn, A.shape[1]) if need_dS0 else (0,)))


# The short causal convolution:
#     y, state = torch.ops.subq_audio.causal_conv_fwd(x, weight, bias, mask, state, activation, want_state)
#     dx, dweight, dbias, dstate = torch.ops.subq_audio.causal_conv_bwd(x, weight, dout, bias, mask, state, dstate, activation, need_dstate)
@torch.library.custom_op("subq_audio::causal_conv_fwd", mutates_args=(), device_types="cuda")
def causal_conv_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], mask: Optional[Tensor], state: Optional[Tensor], activation: Optional[str],
                    want_state: bool) -> Tuple[Tensor, Tensor]:
    y, S = ops.causal_conv_forward(x, weight, bias, activation=activation, mask=mask, state=state, return_state=want_state)
    return y, (S if want_state else x.new_empty(0))


@causal_conv_fwd.register_fake
def _causal_conv_fwd_fake(x, weight, bias, mask, state, activation, want_state):
    S = x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2]) if want_state else (0,))
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), S


@torch.library.custom_op("subq_audio::causal_conv_bwd", mutates_args=(), device_types="cuda")
def causal_conv_bwd(x: Tensor, weight: Tensor, dout: Tensor, bias: Optional[Tensor], mask: Optional[Tensor], state: Optional[Tensor],
                    dstate: Optional[Tensor], activation: Optional[str], need_dstate: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    dx, dw, db, ds = ops.causal_conv_backward(x, weight, dout, bias, activation=activation, mask=mask, state=state, dstate=dstate, need_dstate=need_dstate)
    return dx, dw, (db if db is not None else _empty_f32(x, (0,))), (ds if ds is not None else x.new_empty(0))


@causal_conv_bwd.register_fake
def _causal_conv_bwd_fake(x, weight, dout, bias, mask, state, dstate, activation, need_dstate):
    D, W = weight.shape
    return (torch.empty(x.shape, dtype=x.dtype, device=x.device), _empty_f32(x, (D, W)), _empty_f32(x, (0 if bias is None else D,)),
            x.new_empty((x.shape[0], W - 1, D) if need_dstate else (0,)))


# RMSNorm with a residual's addition (r is empty without one), and its gradients from r (dx is empty where it is dres):
#     y, r = torch.ops.subq_audio.rms_norm_fwd(x, weight, residual, eps, out_dtype)
#     dres, dx, dweight = torch.ops.subq_audio.rms_norm_bwd(dy, r, weight, dr, eps, need_dweight)
@torch.library.custom_op("subq_audio::rms_norm_fwd", mutates_args=(), device_types="cuda")
def rms_norm_fwd(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float, out_dtype: Optional[torch.dtype]) -> Tuple[Tensor, Tensor]:
    got = ops.rms_norm(x, weight, eps, residual=residual, out_dtype=out_dtype)
    return got if residual is not None else (got, x.new_empty(0))


@rms_norm_fwd.register_fake
def _rms_norm_fwd_fake(x, weight, residual, eps, out_dtype):
    r = x.new_empty(0) if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    return torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device), r


@torch.library.custom_op("subq_audio::rms_norm_bwd", mutates_args=(), device_types="cuda")
def rms_norm_bwd(dy: Tensor, r: Tensor, weight: Optional[Tensor], dr: Optional[Tensor], eps: float, need_dweight: bool) -> Tuple[Tensor, Tensor, Tensor]:
    dx, dres, dw = ops.rms_norm_backward(dy, r, weight, eps, dresidual=dr, need_dweight=need_dweight)
    return dres, (dx if dx is not dres else dy.new_empty(0)), (dw if dw is not None else _empty_f32(r, (0,)))


@rms_norm_bwd.register_fake
def _rms_norm_bwd_fake(dy, r, weight, dr, eps, need_dweight):
    dres = torch.empty(r.shape, dtype=r.dtype, device=r.device)
    dx = dy.new_empty(0) if dy.dtype == r.dtype else torch.empty(r.shape, dtype=dy.dtype, device=r.device)
    return dres, dx, _empty_f32(r, (r.shape[-1] if need_dweight else 0,))


# The 8-bit forms (for inference: no gradients):
#     q, scale, r = torch.ops.subq_audio.rms_norm_fp8(x, weight, residual, eps)
#     q, scale = torch.ops.subq_audio.quantize_fp8(x)
#     out = torch.ops.subq_audio.scaled_matmul(a, a_scale, b, b_scale, bias, out_dtype)
def _fp8_fake(x):
    q, scale = ops.block_ops._fp8_rows(x)
    return q, scale


@torch.library.custom_op("subq_audio::rms_norm_fp8", mutates_args=(), device_types="cuda")
def rms_norm_fp8(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    got = ops.rms_norm_fp8(x, weight, eps, residual=residual)
    return got if residual is not None else (*got, x.new_empty(0))


@rms_norm_fp8.register_fake
def _rms_norm_fp8_fake(x, weight, residual, eps):
    return (*_fp8_fake(x), x.new_empty(0) if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device))


@torch.library.custom_op("subq_audio::quantize_fp8", mutates_args=(), device_types="cuda")
def quantize_fp8(x: Tensor) -> Tuple[Tensor, Tensor]:
    return ops.quantize_fp8(x)


@quantize_fp8.register_fake
def _quantize_fp8_fake(x):
    return _fp8_fake(x)


@torch.library.custom_op("subq_audio::scaled_matmul", mutates_args=(), device_types="cuda")
def scaled_matmul(a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor, bias: Optional[Tensor], out_dtype: torch.dtype) -> Tensor:
    return ops.scaled_matmul(a, a_scale, b, b_scale, bias=bias, out_dtype=out_dtype)


@scaled_matmul.register_fake
def _scaled_matmul_fake(a, a_scale, b, b_scale, bias, out_dtype):
    return torch.empty((*a.shape[:-1], b.shape[0]), dtype=out_dtype, device=a.device)
