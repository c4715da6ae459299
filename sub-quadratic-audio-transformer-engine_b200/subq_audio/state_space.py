"""A selective state space layer on the kernels: differentiable calls and modules.

``selective_scan`` and ``causal_conv`` stand beside ``gated_delta_attention`` and ``chunkwise_flash_linear_attention``: a third
recurrence over [B, L, *] sequences with the same masks, carried state and ``past_key_values`` threading. ``rms_norm`` is the
norm before such a layer with the residual's addition in it. ``SubQSelectiveStateSpace`` is the layer (``SubQLinearAttention``'s
call contract), ``SubQStateSpaceBlock`` the norm and the layer; ``quantize`` turns their projections into 8-bit ones for
inference (``SubQFp8Linear``), which read the norm's 8-bit output as it is.
"""
from __future__ import annotations

import math
from typing import Any, Optional, Tuple, Union

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import library as _library  # noqa: F401  (registers torch.ops.subq_audio)
from .autograd import _normalize_attention_mask, _split_state, _token_mask

Pair = Tuple[torch.Tensor, torch.Tensor]


def _mask_of(attention_mask: Optional[torch.Tensor], x: torch.Tensor) -> Optional[torch.Tensor]:
    if attention_mask is None:
        return None
    if attention_mask.dtype in (torch.bool, torch.uint8) and attention_mask.shape == x.shape[:2] and attention_mask.device == x.device:
        return attention_mask
    valid = _normalize_attention_mask(attention_mask.to(x.device), x.dtype, x.shape[1])
    return _token_mask(valid, x.shape[0], x.shape[1], x.device)


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in ts)


def _to(g: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return g.to(like.dtype)


class _SelectiveScan(torch.autograd.Function):
    """The scan on the kernels; differentiable in every input and through the states. The forward keeps its handover for the
    backward where one will follow (``ops.ScanHandover`` has its size)."""

    @staticmethod
    def forward(ctx, u, dt, A, B, C, D, z, dt_bias, mask, S0, dt_softplus, want_state, keep):
        y, S, handover = torch.ops.subq_audio.selective_scan_fwd(u, dt, A, B, C, D, z, dt_bias, mask, S0, dt_softplus, want_state, keep)
        ctx.softplus, ctx.want_state = dt_softplus, want_state
        ctx.save_for_backward(u, dt, A, B, C, D, z, dt_bias, mask, S0, handover)
        ctx.set_materialize_grads(False)
        return (y, S) if want_state else (y, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dS):
        u, dt, A, B, C, D, z, dt_bias, mask, S0, handover = ctx.saved_tensors
        if dy is None and dS is None:
            return (None,) * 13
        need = ctx.needs_input_grad
        need_S0 = S0 is not None and need[9]
        dy = torch.zeros_like(u) if dy is None else dy.to(u.dtype)
        du, ddt, dA, dB, dC, dD, dz, dbias, dS0 = torch.ops.subq_audio.selective_scan_bwd(
            u, dt, A, B, C, dy, D, z, dt_bias, mask, S0, dS, ctx.softplus, handover, need_S0)
        return (du, ddt, _to(dA, A) if need[2] else None, dB, dC, _to(dD, D) if D is not None and need[5] else None, dz if z is not None else None,
                _to(dbias, dt_bias) if dt_bias is not None and need[7] else None, None, _to(dS0, S0) if need_S0 else None, None, None, None)


def selective_scan(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = True, past_state: Any = None,
                   attention_mask: Optional[torch.Tensor] = None, return_state: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The selective scan, differentiable (``ops.selective_scan_forward`` has the formula and the shapes). ``past_state`` is a
    state [B, D, N] or a tuple that starts with one; ``attention_mask`` as in ``chunkwise_flash_linear_attention``. Returns
    ``(out, S_next)``; gradients also flow through the states. Of first order and reverse mode (second gradients, forward
    mode and ``torch.func`` transforms raise)."""
    S0 = None if past_state is None else _split_state(past_state)[0]
    keep = _wants_grad(u, dt, A, B, C, D, z, dt_bias, S0)
    return _SelectiveScan.apply(u, dt, A, B, C, D, z, dt_bias, _mask_of(attention_mask, u), S0, dt_softplus, return_state, keep)


class _CausalConv(torch.autograd.Function):
    """The short convolution on the kernels; saves its inputs (the backward forms the sums before the activation again)."""

    @staticmethod
    def forward(ctx, x, weight, bias, mask, state, activation, want_state):
        y, S = torch.ops.subq_audio.causal_conv_fwd(x, weight, bias, mask, state, activation, want_state)
        ctx.activation, ctx.want_state = activation, want_state
        ctx.save_for_backward(x, weight, bias, mask, state)
        ctx.set_materialize_grads(False)
        return (y, S) if want_state else (y, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dS):
        x, weight, bias, mask, state = ctx.saved_tensors
        if dy is None and dS is None:
            return (None,) * 7
        need_S = state is not None and ctx.needs_input_grad[4]
        dy = torch.zeros_like(x) if dy is None else dy.to(x.dtype)
        dx, dw, db, ds = torch.ops.subq_audio.causal_conv_bwd(x, weight, dy, bias, mask, state, dS, ctx.activation, need_S)
        return (dx, _to(dw, weight) if ctx.needs_input_grad[1] else None, _to(db, bias) if bias is not None and ctx.needs_input_grad[2] else None, None,
                _to(ds, state) if need_S else None, None, None)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
                past_state: Optional[torch.Tensor] = None, attention_mask: Optional[torch.Tensor] = None, return_state: bool = True
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The short causal convolution, differentiable (``ops.causal_conv_forward``): ``(y, window)``; ``past_state`` and the
    returned window are [B, W - 1, D]. Of first order and reverse mode."""
    return _CausalConv.apply(x, weight, bias, _mask_of(attention_mask, x), past_state, activation, return_state)


class _RMSNorm(torch.autograd.Function):
    """RMSNorm with a residual's addition; saves r alone (x without a residual)."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, out_dtype):
        y, r = torch.ops.subq_audio.rms_norm_fwd(x, weight, residual, eps, out_dtype)
        ctx.eps, ctx.types = eps, (x.dtype, None if weight is None else weight.dtype)
        ctx.has_residual = residual is not None
        ctx.save_for_backward(r if residual is not None else x, weight)
        ctx.set_materialize_grads(False)
        return (y, r) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr=None):
        r, weight = ctx.saved_tensors
        x_type, w_type = ctx.types
        need_w = weight is not None and ctx.needs_input_grad[1]
        if dy is None:  # the residual stream's gradient alone
            if dr is None:
                return (None,) * 5
            return dr.to(x_type), (torch.zeros_like(weight) if need_w else None), dr, None, None
        dres, dx, dw = torch.ops.subq_audio.rms_norm_bwd(dy, r, weight, None if dr is None else dr.to(r.dtype), ctx.eps, need_w)
        dx = dx if dx.numel() and dx.dtype == x_type else dres.to(x_type)
        return dx, dw.to(w_type) if need_w else None, dres if ctx.has_residual else None, None, None


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5, residual: Optional[torch.Tensor] = None,
             out_dtype: Optional[torch.dtype] = None):
    """RMSNorm over the last dimension with a residual's addition before it, differentiable once, in reverse mode
    (``ops.rms_norm``): ``y``, or ``(y, r)`` with a residual."""
    return _RMSNorm.apply(x, weight, residual, eps, out_dtype)


class SubQRMSNorm(nn.Module):
    """RMSNorm on the kernels: ``norm(x)`` is y, ``norm(x, residual)`` is (y, r) with r = x + residual, the residual stream that
    goes on. As with ``SubQLayerNorm``, a float32 input under autocast gives the autocast type (``out_dtype`` for another)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None):
        super().__init__()
        if not 1 <= hidden_size <= 16384:
            raise ValueError(f"the norm's kernels take 1 to 16384 columns, got {hidden_size}")
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.eps, self.out_dtype = eps, out_dtype

    def _out(self, x: torch.Tensor) -> torch.dtype:
        if x.dtype != torch.float32:
            return x.dtype
        if self.out_dtype is not None:
            return self.out_dtype
        return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, self.eps, residual, self._out(x))

    def quantized(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """``(q, scale)`` in 8 bits, or ``(q, scale, r)``: what ``SubQFp8Linear`` reads. For inference."""
        q, scale, r = torch.ops.subq_audio.rms_norm_fp8(x, self.weight, residual, self.eps)
        return (q, scale) if residual is None else (q, scale, r)


class SubQFp8Linear(nn.Module):
    """A linear layer's weight in 8 bits with a float32 scale for every 128 x 128 of it, for inference. Takes a tensor (made 8 bits
    wide with a scale for every 128 of a row) or such a pair ``(q, scale)`` as it is. ``out_dtype`` is the result's type for
    pairs, a tensor's result has its type, and a call's own ``out_dtype`` comes before both. The 8-bit weight and its scales are
    kept as bytes, so that casting the module leaves them alone."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, out_dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if not 1 <= in_features <= 16384 or out_features < 1:
            raise ValueError(f"the 8-bit layer takes 1 to 16384 columns and at least a row, got {in_features} and {out_features}")
        self.in_features, self.out_features, self.out_dtype = in_features, out_features, out_dtype
        n, k = (out_features + 127) // 128, (in_features + 127) // 128
        self.register_buffer("weight_bytes", torch.zeros(out_features, (in_features + 15) // 16 * 16, dtype=torch.uint8, device=device))
        self.register_buffer("scale_bytes", torch.zeros(n, 4 * k, dtype=torch.uint8, device=device))
        self.register_buffer("bias", torch.zeros(out_features, device=device) if bias else None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear, out_dtype: Optional[torch.dtype] = None) -> "SubQFp8Linear":
        from . import ops

        w = linear.weight
        if out_dtype is None:
            out_dtype = w.dtype if w.dtype in (torch.float16, torch.bfloat16) else torch.bfloat16
        new = cls(linear.in_features, linear.out_features, linear.bias is not None, out_dtype, w.device)
        q, scale = ops.quantize_fp8_weight(w)
        new.weight_bytes[:, :linear.in_features] = q.view(torch.uint8)
        new.scale_bytes.copy_(scale.view(torch.uint8))
        if linear.bias is not None:
            new.bias.copy_(linear.bias)
        return new

    def forward(self, x: Union[torch.Tensor, Pair], out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        if isinstance(x, tuple):
            (q, scale), out = x, out_dtype or self.out_dtype
        else:
            if _wants_grad(x):
                raise RuntimeError("SubQFp8Linear is for inference: it has no gradients")
            q, scale = torch.ops.subq_audio.quantize_fp8(x)
            out = out_dtype or x.dtype
        w = self.weight_bytes.view(torch.float8_e4m3fn)[:, :self.in_features]
        return torch.ops.subq_audio.scaled_matmul(q, scale, w, self.scale_bytes.view(torch.float32), self.bias, out)


class SubQSelectiveStateSpace(nn.Module):
    """A selective state space layer with ``SubQLinearAttention``'s call contract: one projection into a branch and its gate, the
    short causal convolution of the branch, step sizes, B and C projected from it, the selective scan with the gate, one
    projection out. Causal. ``past_state`` and the returned state are the scan's [B, inner, N] float32 with the
    convolution's last inputs [B, W - 1, inner] attached as ``.Z`` (or the pair of them), so that ``cache.run_layers`` and
    ``StateCache`` thread them. ``quantize()`` makes the outer projections 8 bits wide, for inference."""

    def __init__(self, hidden_size: int, expand: int = 2, state_size: int = 16, conv_width: int = 4, dt_rank: Optional[int] = None, groups: int = 1,
                 dt_min: float = 0.001, dt_max: float = 0.1, bias: bool = False, conv_bias: bool = True):
        super().__init__()
        inner = expand * hidden_size
        if not 1 <= state_size <= 128:
            raise ValueError(f"the scan's kernels take 1 to 128 states a channel, got {state_size}")
        if not 2 <= conv_width <= 4:
            raise ValueError(f"the convolution's kernels take a width of 2, 3 or 4, got {conv_width}")
        if groups < 1 or inner % groups:
            raise ValueError(f"{inner} channels do not divide into {groups} groups")
        if not 0 < dt_min <= dt_max:
            raise ValueError("step sizes need 0 < dt_min <= dt_max")
        # (a multiple of 8, so that B and C start on 16-byte boundaries behind it)
        self.dt_rank = dt_rank if dt_rank is not None else max(8, (hidden_size // 16 + 7) // 8 * 8)
        self.hidden_size, self.inner, self.state_size, self.groups = hidden_size, inner, state_size, groups
        self.in_proj = nn.Linear(hidden_size, 2 * inner, bias=bias)
        self.conv_weight = nn.Parameter(torch.empty(inner, conv_width))
        self.conv_bias = nn.Parameter(torch.zeros(inner)) if conv_bias else None
        self.x_proj = nn.Linear(inner, self.dt_rank + 2 * groups * state_size, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, inner, bias=False)
        nn.init.uniform_(self.conv_weight, -conv_width ** -0.5, conv_width ** -0.5)
        nn.init.uniform_(self.dt_proj.weight, -self.dt_rank ** -0.5, self.dt_rank ** -0.5)
        # step sizes between dt_min and dt_max, evenly over their logarithm: softplus(dt_bias)
        size = torch.exp(torch.rand(inner) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
        self.dt_bias = nn.Parameter(size + torch.log(-torch.expm1(-size)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, state_size + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, hidden_size, bias=bias)

    def quantize(self) -> "SubQSelectiveStateSpace":
        for name in ("in_proj", "out_proj"):
            if isinstance(getattr(self, name), nn.Linear):
                setattr(self, name, SubQFp8Linear.from_linear(getattr(self, name)))
        return self

    def forward(self, hidden_states: Union[torch.Tensor, Pair], past_state: Any = None, attention_mask: Optional[torch.Tensor] = None,
                use_cache: bool = False, **kwargs: Any):
        S0 = window = None
        if past_state is not None:
            S0, window = _split_state(past_state)
            if window is None:
                raise ValueError("past_state needs the scan's state and the convolution's window (state.Z, or a pair)")
        if isinstance(hidden_states, tuple):  # (8 bits say nothing of the branch's type: what the next projection takes)
            branch = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else self.x_proj.weight.dtype
            xz = self.in_proj(hidden_states, branch)
        else:
            xz = self.in_proj(hidden_states)
        x, z = xz[..., :self.inner], xz[..., self.inner:]
        mask = _mask_of(attention_mask, x)
        x, window = causal_conv(x, self.conv_weight, self.conv_bias, "silu", None if window is None else window.to(x.dtype), mask, use_cache)
        p = self.x_proj(x)
        R, GN = self.dt_rank, self.groups * self.state_size
        B, C = (p[..., i:i + GN].unflatten(-1, (self.groups, self.state_size)) for i in (R, R + GN))
        x, dt, B, C, z = _one_type(x, self.dt_proj(p[..., :R]), B, C, z)
        y, S = selective_scan(x, dt, -torch.exp(self.A_log.float()), B, C, self.D, z, self.dt_bias, True, S0, mask, use_cache)
        out = self.out_proj(y)
        if not use_cache:
            return out, None
        S.Z = window
        return out, S


def _one_type(x: torch.Tensor, *others: torch.Tensor):
    return (x,) + tuple(t if t.dtype == x.dtype else t.to(x.dtype) for t in others)


class SubQStateSpaceBlock(nn.Module):
    """RMSNorm and ``SubQSelectiveStateSpace`` around a residual stream, the addition inside the norm: takes a tensor (the stream,
    at the first block) or the pair ``(branch, stream)`` that the block before returned, and returns
    ``((branch, stream), state)``, as ``cache.run_layers`` threads it; ``norm(branch, stream)`` of a last ``SubQRMSNorm`` closes a
    stack. Quantised and without gradients, the norm gives its 8-bit output to the projection."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, **layer: Any):
        super().__init__()
        self.norm = SubQRMSNorm(hidden_size, eps)
        self.mixer = SubQSelectiveStateSpace(hidden_size, **layer)

    def quantize(self) -> "SubQStateSpaceBlock":
        self.mixer.quantize()
        return self

    def forward(self, hidden_states: Union[torch.Tensor, Pair], past_state: Any = None, attention_mask: Optional[torch.Tensor] = None,
                use_cache: bool = False, **kwargs: Any):
        x, stream = hidden_states if isinstance(hidden_states, tuple) else (hidden_states, None)
        if isinstance(self.mixer.in_proj, SubQFp8Linear):
            if _wants_grad(x, stream, self.norm.weight):
                raise RuntimeError("a quantised block is for inference: it has no gradients")
            q, scale, *r = self.norm.quantized(x, stream)
            out, state = self.mixer((q, scale), past_state, attention_mask, use_cache)
        else:
            got = self.norm(x, stream)
            h, *r = got if stream is not None else (got,)
            out, state = self.mixer(h, past_state, attention_mask, use_cache)
        return (out, r[0] if r else x), state
