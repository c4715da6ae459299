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
