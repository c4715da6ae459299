"""The gated delta rule and layer norm as differentiable calls and modules.

``gated_delta_attention`` and ``SubQGatedDeltaAttention`` stand beside
``chunkwise_flash_linear_attention`` and ``SubQLinearAttention``: the same
shapes, masks, grouped K/V, carried state and ``past_key_values`` threading
(``cache.run_layers``, ``StateCache``), with an update that corrects what the
state holds for a key instead of adding to it:

    S_t = gamma_t S_{t-1} + beta_t k_t (v_t - gamma_t S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t

``layer_norm`` and ``SubQLayerNorm`` are the norm before such a layer.
"""
from __future__ import annotations

import math
from typing import Any, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import library as _library  # noqa: F401  (registers torch.ops.subq_audio)
from . import ops
from .autograd import (_HeadRMSNorm, _normalize_attention_mask, _split_state, _to_device_inputs, _token_mask,
                       apply_rotary_pos_emb)


def _strided(x: Optional[torch.Tensor]) -> bool:
    return x is not None and x.dim() == 3 and not x.is_contiguous()


def _gate_grad(g: Optional[torch.Tensor], x: Optional[torch.Tensor], strided: bool) -> Optional[torch.Tensor]:
    """The per-token gradient [B, H, N] in the shape and type of the gate x ([], [H] or broadcastable)."""
    if g is None or x is None:
        return None
    if x.dim() == 1:
        g = g.sum(dim=(0, 2))
    else:
        g = g.sum_to_size(x.shape)
    if strided:
        # in the gate's own memory order (a [B, H, N] view of a projection's [B, N, H] output): the elementwise
        # operations that follow then see one layout, traced or not
        return torch.empty_like(x).copy_(g)
    return g.to(x.dtype)


class _GatedDelta(torch.autograd.Function):
    """The rule on the kernels; differentiable in q, k, v, beta, log_gamma and the initial state, and through the
    final state. The forward keeps its handover for the backward where one will follow (``ops.DeltaHandover`` has its
    size; ``torch.utils.checkpoint`` around the layer keeps it from staying)."""

    @staticmethod
    def forward(ctx, q, k, v, beta, lg, mask, S0, scale, want_state, keep):
        o, S, handover = torch.ops.subq_audio.gated_delta_fwd(q, k, v, beta, lg, mask, S0, scale, want_state, keep)
        ctx.scale, ctx.want_state = scale, want_state
        ctx.strided = (_strided(beta), _strided(lg))
        ctx.save_for_backward(q, k, v, beta, lg, mask, S0, handover)
        ctx.set_materialize_grads(False)
        return (o, S) if want_state else (o, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dS):
        q, k, v, beta, lg, mask, S0, handover = ctx.saved_tensors
        if do is None:
            if dS is None:
                return (None,) * 10
            H = dS.shape[1]
            do = q.new_zeros(q.shape[0], H, q.shape[2], v.shape[-1])
        need_lg = lg is not None and ctx.needs_input_grad[4]
        need_S0 = S0 is not None and ctx.needs_input_grad[6]
        dq, dk, dv, dbeta, dlg, dS0 = torch.ops.subq_audio.gated_delta_bwd(
            q, k, v, beta, do, lg, mask, S0, dS, ctx.scale, handover, need_lg, need_S0)
        return (dq, dk, dv, _gate_grad(dbeta, beta, ctx.strided[0]) if ctx.needs_input_grad[3] else None,
                _gate_grad(dlg, lg, ctx.strided[1]) if need_lg else None, None, dS0.to(S0.dtype) if need_S0 else None, None, None, None)


def gated_delta_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: Any, log_gamma: Any = None,
                          past_state: Any = None, attention_mask: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None, return_state: bool = True
                          ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The gated delta rule, differentiable (``ops.gated_delta_forward`` has the formula and the head layout).

    ``q``, ``k``, ``v`` are [B, T, D] or [B, H, T, D]; ``beta`` and ``log_gamma`` (log of the decay, at most 0) are
    None, a number, or a tensor [], [H] or [B, H, T] ([B, T] with 3-D inputs); ``past_state`` a state [B, H, d, e] or a
    tuple that starts with one; ``attention_mask`` as in ``chunkwise_flash_linear_attention``. Returns
    ``(out, S_next)``, out in q's memory order; gradients also flow through the states. The backward needs d <= 128, and is
    of first order and reverse mode (second gradients, forward mode and ``torch.func`` transforms raise).
    """
    is_3d = q.ndim == 3
    if is_3d:
        q, k, v = q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1)
        beta, log_gamma = (g.unsqueeze(1) if isinstance(g, torch.Tensor) and g.ndim == 2 else g for g in (beta, log_gamma))
    q, k, v, home = _to_device_inputs(q, k, v)
    B, _, T, d = q.shape
    beta, log_gamma = (g if g is None else g.to(q.device) if isinstance(g, torch.Tensor) else
                       torch.full((), float(g), dtype=torch.float32, device=q.device) for g in (beta, log_gamma))
    valid = _normalize_attention_mask(attention_mask.to(q.device) if attention_mask is not None else None, q.dtype, T)
    mask = _token_mask(valid, B, T, q.device)
    S0 = None
    if past_state is not None:
        S0 = _split_state(past_state)[0].to(q.device)
    keep = torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v, beta, log_gamma, S0))
    out, S = _GatedDelta.apply(q, k, v, beta, log_gamma, mask, S0, d ** -0.5 if scale is None else float(scale), return_state, keep)
    if is_3d:
        out = out.squeeze(1)
    if home is not None:
        out = out.to(home)
    return out, S


class _LayerNorm(torch.autograd.Function):
    """Layer norm on the kernels; saves x alone (the backward recomputes the statistics)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        ctx.types = (weight.dtype if weight is not None else None, bias.dtype if bias is not None else None)
        return torch.ops.subq_audio.layer_norm_fwd(x, weight, bias, eps, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        dx, dw, db = torch.ops.subq_audio.layer_norm_bwd(dy, x, weight, ctx.eps, need_w, need_b)
        return dx, dw.to(ctx.types[0]) if need_w else None, db.to(ctx.types[1]) if need_b else None, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Layer norm over the last dimension, differentiable once, in reverse mode (``ops.layer_norm``). ``torch.func``
    transforms, forward mode and second gradients raise: torch's ``layer_norm`` has them."""
    return _LayerNorm.apply(x, weight, bias, eps, out_dtype)


class SubQLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension on the library's kernels. Under autocast a float32 input gives the
    autocast type (the layer that follows reads its 16-bit input as it is; torch's norm returns float32, cast again
    for each projection); where something else than a projection follows, ``out_dtype=torch.float32`` keeps torch's
    result. ``out_dtype`` holds for float32 inputs, with or without autocast; a 16-bit input gives its own type. Inputs
    the kernels do not take (CPU, float64, several dimensions, another width) go to torch's norm. The gradient is
    ``layer_norm``'s: first order, reverse mode (no second gradients, forward mode or ``torch.func`` transforms)."""

    out_dtype: Optional[torch.dtype] = None

    def __init__(self, *args: Any, out_dtype: Optional[torch.dtype] = None, **kwargs: Any):
        super().__init__(*args, **kwargs)
        self.out_dtype = out_dtype

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if (not x.is_cuda or len(self.normalized_shape) != 1 or x.shape[-1:] != self.normalized_shape
                or x.dtype not in (torch.float32, torch.float16, torch.bfloat16)):
            return super().forward(x)
        out = x.dtype
        if x.dtype == torch.float32:
            if self.out_dtype is not None:
                out = self.out_dtype
            elif torch.is_autocast_enabled("cuda"):
                out = torch.get_autocast_dtype("cuda")
        return layer_norm(x, self.weight, self.bias, self.eps, out)


class SubQGatedDeltaAttention(nn.Module):
    """A gated-delta layer with ``SubQLinearAttention``'s call contract: q/k/v/out projections, optional rotary
    positions, grouped K/V, queries and keys scaled to unit length per head, beta = sigmoid of a projection, decay
    = sigmoid(raw_decay + projection) per token and head, per-head RMSNorm of the output. Causal only. ``past_state``
    and the returned state are [B, H, D, D] float32; single tokens run the token-recurrent kernel. Heads of at most 256
    dimensions; of at most 128 where the layer is trained (the kernels have no backward above)."""

    def __init__(self, hidden_size: int, num_heads: int = 1, num_key_value_heads: Optional[int] = None,
                 decay_init: float = 0.99, bias: bool = False):
        super().__init__()
        self.hidden_size, self.num_heads = hidden_size, num_heads
        self.num_key_value_heads = num_key_value_heads if num_key_value_heads is not None else num_heads
        self.head_dim = hidden_size // num_heads
        if self.head_dim * num_heads != hidden_size:
            raise ValueError(f"hidden_size {hidden_size} must be divisible by num_heads {num_heads}")
        if self.num_heads % self.num_key_value_heads != 0:
            raise ValueError(f"num_heads {num_heads} must be divisible by num_key_value_heads {self.num_key_value_heads}")
        if self.head_dim > 256:
            raise ValueError(f"heads of {self.head_dim} dimensions are wider than the kernels' 256: more heads are needed")
        kv = self.num_key_value_heads * self.head_dim
        self.q_proj = nn.Linear(hidden_size, hidden_size, bias=bias)
        self.k_proj = nn.Linear(hidden_size, kv, bias=bias)
        self.v_proj = nn.Linear(hidden_size, kv, bias=bias)
        self.beta_proj = nn.Linear(hidden_size, num_heads, bias=bias)
        self.gate_proj = nn.Linear(hidden_size, num_heads, bias=bias)
        self.out_proj = nn.Linear(hidden_size, hidden_size, bias=bias)
        self.head_norm = nn.RMSNorm(self.head_dim, eps=1e-5)
        d0 = min(max(decay_init, 1e-4), 1.0 - 1e-4)
        self.raw_decay = nn.Parameter(torch.full((num_heads,), math.log(d0 / (1.0 - d0)), dtype=torch.float32))
        # x / sqrt(|x|^2 + 1e-6) is the per-head RMSNorm kernel with this weight
        self.register_buffer("unit", torch.full((self.head_dim,), self.head_dim ** -0.5), persistent=False)

    def _unit_heads(self, x: torch.Tensor) -> torch.Tensor:
        if ops.head_rmsnorm_supported(x):
            return _HeadRMSNorm.apply(x, self.unit, 1e-6 / self.head_dim)
        y = x.float()  # a width the kernel does not take: the same function
        return (y * torch.rsqrt(y.square().sum(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, hidden_states: torch.Tensor, past_state: Any = None, attention_mask: Optional[torch.Tensor] = None,
                use_cache: bool = False, position_embeddings: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, **kwargs: Any):
        B, L, _ = hidden_states.shape

        def heads(x):
            return x.view(B, L, -1, self.head_dim).transpose(1, 2)

        q, k, v = heads(self.q_proj(hidden_states)), heads(self.k_proj(hidden_states)), heads(self.v_proj(hidden_states))
        if position_embeddings is not None:
            q, k = apply_rotary_pos_emb(q, k, *position_embeddings)
            q, k = q.to(v.dtype), k.to(v.dtype)
        q, k = self._unit_heads(q), self._unit_heads(k)
        beta = torch.sigmoid(self.beta_proj(hidden_states).float()).transpose(1, 2)
        log_gamma = -F.softplus(-(self.raw_decay + self.gate_proj(hidden_states).float())).transpose(1, 2)
        # (q and k of unit length: scale 1, as the RMSNorm that follows takes any scale out but for its eps)
        out, state = gated_delta_attention(q, k, v, beta, log_gamma, past_state, attention_mask, scale=1.0, return_state=use_cache)
        if ops.head_rmsnorm_supported(out):
            out = _HeadRMSNorm.apply(out, self.head_norm.weight, self.head_norm.eps)
        else:
            out = self.head_norm(out.float()).to(out.dtype)
        return self.out_proj(out.transpose(1, 2).reshape(B, L, self.hidden_size)), (state if use_cache else None)
