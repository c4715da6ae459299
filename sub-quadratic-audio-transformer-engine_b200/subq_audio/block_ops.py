"""Launchers of a selective state space block's kernels (through the C ABI): the selective scan, the short causal
convolution before it, the residual RMSNorm and the 8-bit projections. ``ops`` exports them.

Sequences are [B, L, D] CUDA tensors (any strides with a contiguous last dimension), as a projection gives them. As in
``ops``: computation is stream-ordered on torch's current stream, nothing synchronises, CPU tensors raise.
"""
from __future__ import annotations

import ctypes
import functools
import inspect
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _capi
from .ops import _DTYPES, _inner_contig, _require_cuda, _workspace

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_E4M3 = torch.float8_e4m3fn
_BLOCK = 128


try:  # (the handle alone, without the object around it: a third of a short call's host time)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


def _stream(device: torch.device) -> int:
    return _raw_stream(device.index)


_SIZES: dict = {}  # sizes in bytes that the library gave, by what they depend on


def _size(query, args, *key) -> int:
    """query(args), asked for once for each key (the call's sizes, which alone it depends on)."""
    n = _SIZES.get((query, key))
    if n is None:
        n = query(args)
        if n:  # (0 may also be the answer to arguments that the call will refuse)
            if len(_SIZES) > 4096:
                _SIZES.clear()
            _SIZES[(query, key)] = n
    return n


def _on_its_device(call):
    """The call with the device of its first tensor as the current one."""
    name = next(iter(inspect.signature(call).parameters))

    @functools.wraps(call)
    def run(*args, **kwargs):
        first = args[0] if args else kwargs.get(name)
        if not (isinstance(first, torch.Tensor) and first.is_cuda):
            if not args and name not in kwargs:
                return call(*args, **kwargs)  # (refuses by itself)
            _require_cuda(first)
        index = first.get_device()
        if index == torch.cuda.current_device():
            return call(*args, **kwargs)
        with torch.cuda.device(index):
            return call(*args, **kwargs)

    return run


def _t3(t: Optional[torch.Tensor]) -> _capi.Tensor3:
    """[B, L, *] or [B, L, G, *] with a contiguous last dimension."""
    if t is None:
        return _capi.Tensor3()
    s = t.stride()
    return _capi.Tensor3(t.data_ptr(), s[0], s[1], s[2] if t.dim() == 4 else 0)


def _mask(mask: Optional[torch.Tensor], B: int, L: int, device: torch.device, keep: list) -> Tuple[Optional[int], int]:
    if mask is None:
        return None, 0
    m = mask.detach()
    if m.dim() != 2 or m.shape[0] != B or m.shape[1] != L:
        raise ValueError(f"mask must be [B, L] = [{B}, {L}], got {tuple(m.shape)}")
    if m.device != device:
        raise ValueError("mask must be on the device of the inputs")
    rows = L <= 1 or m.stride(1) == 1  # (one token a row: its place in the row does not matter)
    if m.dtype == torch.bool and rows:
        m = m.view(torch.uint8)
    elif m.dtype != torch.uint8 or not rows:
        m = (m != 0).to(torch.uint8).contiguous()
    keep.append(m)
    return m.data_ptr(), m.stride(0)


def _param(w: Optional[torch.Tensor], name: str, shape: tuple, device: torch.device, keep: list) -> Optional[int]:
    """A float32 parameter's address (converted where it has another type or layout)."""
    if w is None:
        return None
    if w.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(w.shape)}")
    if w.device != device:
        raise ValueError(f"{name} must be on the device of the inputs")
    if w.dtype is not torch.float32 or not w.is_contiguous():
        if not w.is_floating_point():
            raise TypeError(f"{name} must be a floating-point tensor, got {w.dtype}")
        w = w.detach().to(torch.float32).contiguous()
        keep.append(w)
    return w.data_ptr()


def _check_seq(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    if t.shape != like.shape:
        raise ValueError(f"{name} must have shape {tuple(like.shape)}, got {tuple(t.shape)}")
    if t.dtype is not like.dtype:
        raise TypeError(f"{name} must have type {like.dtype}, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} must be on the device {like.device}")


def _check_out(t: torch.Tensor, like: torch.Tensor) -> None:
    _check_seq(t, "out", like)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("out must have a contiguous last dimension")


# ------------------------------------------------------------ causal convolution
def _activation(activation: Optional[str]) -> int:
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return 1 if activation == "silu" else 0


def _conv_args(x, weight, bias, activation, mask, state, keep: list, y: Optional[torch.Tensor] = None, state_out: Optional[int] = None) -> _capi.CausalConvArgs:
    if x.dim() != 3 or weight.dim() != 2:
        raise ValueError("x must be [B, L, D] and weight [D, W]")
    if x.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {x.dtype}; use float32, float16 or bfloat16")
    B, L, D = x.shape
    W = weight.shape[1]
    if not 2 <= W <= 4:
        raise ValueError(f"the convolution's width must be 2, 3 or 4, got {W}")
    dev = x.device
    m, m_stride = (None, 0) if mask is None else _mask(mask, B, L, dev, keep)
    none = _capi.Tensor3()
    return _capi.CausalConvArgs(B, L, D, W, _DTYPES[x.dtype], _activation(activation), _t3(x), none if y is None else _t3(y), none, none,
                                _param(weight, "weight", (D, W), dev, keep), _param(bias, "bias", (D,), dev, keep), m, m_stride,
                                None if state is None else _window(state, "state", x, W, keep), state_out, None, None, None, None, None, 0, _stream(dev))


def _window(state: torch.Tensor, name: str, x: torch.Tensor, W: int, keep: list) -> int:
    shape = (x.shape[0], W - 1, x.shape[2])
    if tuple(state.shape) != shape:
        raise ValueError(f"{name} must be [B, W - 1, D] = {list(shape)}, got {tuple(state.shape)}")
    if state.device != x.device:
        raise ValueError(f"{name} must be on the device of x")
    s = state.detach().to(x.dtype).contiguous()
    keep.append(s)
    return s.data_ptr()


@_on_its_device
def causal_conv_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                        activation: Optional[str] = "silu", mask: Optional[torch.Tensor] = None,
                        state: Optional[torch.Tensor] = None, return_state: bool = False,
                        out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Short causal convolution of [B, L, D], one filter ``weight[d]`` of W = 2, 3 or 4 taps a channel:
    y_t = act(bias + sum_j weight[:, j] x_{t-W+1+j}), act silu or (``activation=None``) nothing. Returns ``(y, state | None)``.

    ``state`` [B, W - 1, D] (x's type) holds the inputs before the first token (None: zeros). A masked token's input counts
    as 0 and its output is 0; nothing of it is used. The returned state is of the W - 1 inputs up to the last live token,
    so that a padded batch of prompts goes on with its next tokens. Math in float32."""
    x = _inner_contig(x)
    keep: list = []
    if out is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        y = out
        _check_out(y, x)
    new = None
    if return_state:
        new = torch.empty((x.shape[0], weight.shape[1] - 1 if weight.dim() == 2 and 2 <= weight.shape[1] <= 4 else 0, x.shape[-1]), dtype=x.dtype, device=x.device)
    _capi.causal_conv_fwd(_conv_args(x, weight, bias, activation, mask, state, keep, y, None if new is None else new.data_ptr()))
    return y, new


@_on_its_device
def causal_conv_backward(x: torch.Tensor, weight: torch.Tensor, dout: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                         activation: Optional[str] = "silu", mask: Optional[torch.Tensor] = None,
                         state: Optional[torch.Tensor] = None, dstate: Optional[torch.Tensor] = None, need_dstate: bool = False
                         ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of ``causal_conv_forward``: ``(dx, dweight, dbias | None, dstate | None)``, dx in x's type, dweight and
    dbias float32. ``dstate`` is the gradient of the returned state (None: 0); with ``need_dstate`` that of ``state`` comes
    back (in x's type)."""
    x, dout = _inner_contig(x), _inner_contig(dout)
    _check_seq(dout, "dout", x)
    keep: list = []
    a = _conv_args(x, weight, bias, activation, mask, state, keep)
    (B, L, D), W, dev = x.shape, weight.shape[1], x.device
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dw = torch.empty((D, W), dtype=torch.float32, device=dev)
    db = ds = None
    a.dy, a.dx, a.dweight = _t3(dout), _t3(dx), dw.data_ptr()
    if bias is not None:
        db = torch.empty(D, dtype=torch.float32, device=dev)
        a.dbias = db.data_ptr()
    if dstate is not None:
        a.dstate_out = _window(dstate, "dstate", x, W, keep)
    if need_dstate:
        ds = torch.empty((B, W - 1, D), dtype=x.dtype, device=dev)
        a.dstate_in = ds.data_ptr()
    a.workspace, a.workspace_bytes = _workspace(_size(_capi.causal_conv_bwd_workspace_bytes, a, B, L, D, W), dev, keep)
    _capi.causal_conv_bwd(a)
    return dx, dw, db, ds


class _Step:
    """One captured argument block over preallocated buffers; ``step()`` enqueues it on the current stream."""

    _run: str

    def _set(self, args, device: torch.device, keep: list) -> None:
        self._args, self.device, self._keep = args, device, keep
        self._call = getattr(_capi.load(), self._run)
        self._ref = ctypes.byref(args)

    def step(self) -> None:
        index = self.device.index
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                return self.step()
        self._args.stream = _raw_stream(index)
        rc = self._call(self._ref)
        if rc:
            _capi.check(rc)


def _own_buffer(t: Optional[torch.Tensor], name: str, shape: tuple, device: torch.device) -> Optional[int]:
    """A step reads the caller's buffers, not copies made at set-up: float32, contiguous."""
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {shape} on the device of the inputs")
    return t.data_ptr()


def _step_mask(mask: Optional[torch.Tensor]) -> None:
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.dim() != 2 or (mask.shape[1] > 1 and mask.stride(1) != 1)):
        raise ValueError("mask must be a bool or uint8 [B, T] tensor with contiguous rows")


def _step_inner(*ts: Optional[torch.Tensor]) -> None:
    if any(t is not None and t.shape[-1] > 1 and t.stride(-1) != 1 for t in ts):
        raise ValueError("the step's buffers must have a contiguous last dimension")


class CausalConvStep(_Step):
    """Streaming form of ``causal_conv_forward`` over preallocated buffers, ``GatedDeltaStep``'s counterpart: ``x`` and
    ``out`` [B, T, D] hold the step's T new tokens (usually 1), ``state`` [B, W - 1, D] (contiguous, x's type) the inputs
    before them; ``weight`` [D, W] and ``bias`` [D] are contiguous float32. ``step()`` writes ``out`` and moves ``state`` on.
    It allocates nothing and does not synchronise, so a CUDA graph can capture it; refill ``x`` in place between steps."""

    _run = "subq_causal_conv_fwd"

    def __init__(self, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], out: torch.Tensor, state: torch.Tensor, *,
                 activation: Optional[str] = "silu", mask: Optional[torch.Tensor] = None):
        _require_cuda(x, weight, out, state)
        _step_inner(x, out)
        _step_mask(mask)
        keep: list = [x, weight, bias, out, state, mask]
        if x.dim() != 3 or weight.dim() != 2:
            raise ValueError("x must be [B, T, D] and weight [D, W]")
        D, W = x.shape[2], weight.shape[1]
        _own_buffer(weight, "weight", (D, W), x.device)
        _own_buffer(bias, "bias", (D,), x.device)
        if state.dtype != x.dtype or not state.is_contiguous() or state.device != x.device:
            raise ValueError(f"state must be a contiguous {x.dtype} tensor on the device of x")
        _check_out(out, x)
        with torch.cuda.device(x.device):
            a = _conv_args(x, weight, bias, activation, mask, state, keep)
            a.state_out = a.state_in
            a.y = _t3(out)
        self._set(a, x.device, keep)


# -------------------------------------------------------------- selective scan
class ScanHandover:
    """Carrier of what ``selective_scan_forward`` leaves for the backward of the same call (the states before every eighth
    token): pass one instance as ``handover=`` to the forward, which fills it, and then to ``selective_scan_backward``, which
    otherwise forms them again. A carrier from a call of another shape, type or device is refused; one from a call of the
    same shape but other inputs gives wrong gradients. It holds 8 bytes for each token and channel of up to 16 states (16,
    32 and 64 bytes up to 32, 64 and 128); without one the backward's workspace holds as much, beside at most 1 GiB or a float32
    [B, L, D] (whichever is more) of parts of dB and dC."""

    def __init__(self) -> None:
        self.buf: Optional[torch.Tensor] = None
        self.key: Optional[tuple] = None


class SelectiveGrads(NamedTuple):
    """What ``selective_scan_backward`` returns: ``dA``, ``dD`` and ``ddt_bias`` float32, ``dstate`` float32, the others in
    the inputs' type and shape; None where there was no such input (``dstate``: where it was not wanted)."""

    du: torch.Tensor
    ddt: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddt_bias: Optional[torch.Tensor]
    dstate: Optional[torch.Tensor]


def _scan_inputs(u, dt, A, B, C, z):
    if u.dim() != 3 or A.dim() != 2:
        raise ValueError("u must be [B, L, D] and A [D, N]")
    if u.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {u.dtype}; use float32, float16 or bfloat16")
    _check_seq(dt, "dt", u)
    if z is not None:
        _check_seq(z, "z", u)
    Bn, L, D = u.shape
    N = A.shape[1]
    if A.shape[0] != D:
        raise ValueError(f"A must be [D, N] with D = {D}, got {tuple(A.shape)}")
    for name, t in (("B", B), ("C", C)):
        if t.dim() not in (3, 4) or t.shape[:2] != u.shape[:2] or t.shape[-1] != N:
            raise ValueError(f"{name} must be [B, L, N] or [B, L, G, N] = [{Bn}, {L}, G, {N}], got {tuple(t.shape)}")
        if t.dtype != u.dtype:
            raise TypeError(f"{name} must have type {u.dtype}, got {t.dtype}")
        if t.device != u.device:
            raise ValueError(f"{name} must be on the device of u")
    if B.shape != C.shape:
        raise ValueError(f"B and C must have one shape, got {tuple(B.shape)} and {tuple(C.shape)}")
    G = B.shape[2] if B.dim() == 4 else 1
    if G < 1 or D % G:
        raise ValueError(f"the {G} groups of B and C must divide the {D} channels")
    if N < 1 or N > 128:
        raise ValueError(f"the scan takes 1 to 128 states a channel, got {N}")
    return G


def _scan_desc(u, A, D, dt_bias, dt_softplus, mask, G: int, keep: list) -> _capi.SelectiveDesc:
    Bn, L, Dn = u.shape
    dev = u.device
    m, m_stride = (None, 0) if mask is None else _mask(mask, Bn, L, dev, keep)
    return _capi.SelectiveDesc(Bn, L, Dn, A.shape[1], G, _DTYPES[u.dtype], 1 if dt_softplus else 0, _param(A, "A", (Dn, A.shape[1]), dev, keep),
                               _param(D, "D", (Dn,), dev, keep), _param(dt_bias, "dt_bias", (Dn,), dev, keep), m, m_stride)


def _state(state: Optional[torch.Tensor], name: str, u: torch.Tensor, N: int, keep: list) -> Optional[int]:
    if state is None:
        return None
    shape = (u.shape[0], u.shape[2], N)
    if tuple(state.shape) != shape:
        raise ValueError(f"{name} must be [B, D, N] = {list(shape)}, got {tuple(state.shape)}")
    if state.device != u.device:
        raise ValueError(f"{name} must be on the device of u")
    s = state.detach().to(torch.float32).contiguous()
    keep.append(s)
    return s.data_ptr()


@_on_its_device
def selective_scan_forward(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                           D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                           dt_softplus: bool = True, mask: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                           return_state: bool = False, out: Optional[torch.Tensor] = None, handover: Optional[ScanHandover] = None
                           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The selective scan. Returns ``(out, state | None)``; the state [B, D, N] is float32.

        dt_t = softplus(dt_t + dt_bias),   h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   out_t = (C_t . h_t + D u_t) silu(z_t)

    ``u``, ``dt``, ``z`` [B, L, D] and ``B``, ``C`` [B, L, N] or [B, L, G, N] (the D / G channels of a group share them)
    have one type (float32, float16 or bfloat16); ``A`` [D, N], ``D`` [D] and ``dt_bias`` [D] are used in float32.
    ``z`` None: no gate; ``dt_softplus=False``: dt + dt_bias itself. ``mask`` [B, L]: a masked token leaves the state as it
    is, its output is 0 and nothing of it is used. N <= 128. Math in float32, a decay near 1 applied as h + (a - 1) h. A raw
    step of -inf (or the type's lowest value) under softplus is a step of 0; one of +inf, as a state or one token's factor exp(dt A) that
    leaves float32's range, leaves infinities or NaN behind, in its channel and from its token on."""
    G = _scan_inputs(u, dt, A, B, C, z)
    u, dt, B, C = (_inner_contig(t) for t in (u, dt, B, C))
    z = None if z is None else _inner_contig(z)
    keep: list = []
    dev, N = u.device, A.shape[1]
    if out is None:
        y = torch.empty(u.shape, dtype=u.dtype, device=dev)
    else:
        y = out
        _check_out(y, u)
    new = None
    if return_state:
        new = torch.empty((u.shape[0], u.shape[2], N), dtype=torch.float32, device=dev)
    a = _capi.SelectiveFwdArgs(_scan_desc(u, A, D, dt_bias, dt_softplus, mask, G, keep), _t3(u), _t3(dt), _t3(z), _t3(B), _t3(C), _t3(y),
                               _state(state, "state", u, N, keep), None if new is None else new.data_ptr(), None, None, 0, _stream(dev))
    sizes = (*u.shape, N, G)
    if handover is not None:
        handover.buf = torch.empty(_size(_capi.selective_scan_handover_bytes, a.desc, *sizes), dtype=torch.uint8, device=dev)
        handover.key = (tuple(u.shape), N, G, u.dtype, dev)
        if handover.buf.numel():
            a.handover = handover.buf.data_ptr()
    nbytes = _size(_capi.selective_scan_fwd_workspace_bytes, a, *sizes, handover is not None)
    if nbytes:
        a.workspace, a.workspace_bytes = _workspace(nbytes, dev, keep)
    _capi.selective_scan_fwd(a)
    return y, new


@_on_its_device
def selective_scan_backward(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, dout: torch.Tensor, *,
                            D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                            dt_softplus: bool = True, mask: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                            dstate: Optional[torch.Tensor] = None, need_dstate: bool = False,
                            handover: Optional[ScanHandover] = None) -> SelectiveGrads:
    """Gradients of ``selective_scan_forward``. ``dstate`` is the gradient of the returned state (None: 0); with
    ``need_dstate`` that of ``state`` comes back. Sums over channels and tokens are float32 in a fixed order: two runs give
    the same bits."""
    G = _scan_inputs(u, dt, A, B, C, z)
    _check_seq(dout, "dout", u)
    u, dt, B, C, dout = (_inner_contig(t) for t in (u, dt, B, C, dout))
    z = None if z is None else _inner_contig(z)
    keep: list = []
    dev, N, (Bn, L, Dn) = u.device, A.shape[1], u.shape

    def like(t):
        return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=dev)

    def f32(*shape):
        return torch.empty(shape, dtype=torch.float32, device=dev)

    g = SelectiveGrads(like(u), like(dt), f32(Dn, N), like(B), like(C), None if D is None else f32(Dn), like(z),
                       None if dt_bias is None else f32(Dn), f32(Bn, Dn, N) if need_dstate else None)
    at = [None if t is None else t.data_ptr() for t in (g.dstate, g.dA, g.dD, g.ddt_bias)]
    a = _capi.SelectiveBwdArgs(_scan_desc(u, A, D, dt_bias, dt_softplus, mask, G, keep), _t3(u), _t3(dt), _t3(z), _t3(B), _t3(C), _t3(dout), _t3(g.du),
                               _t3(g.ddt), _t3(g.dz), _t3(g.dB), _t3(g.dC), _state(state, "state", u, N, keep), _state(dstate, "dstate", u, N, keep), *at,
                               None, None, 0, _stream(dev))
    sizes = (Bn, L, Dn, N, G)
    handed = handover is not None and handover.buf is not None and handover.buf.numel() > 0
    if handed:
        if handover.key != (tuple(u.shape), N, G, u.dtype, dev):
            raise ValueError("handover comes from a forward of another shape, type or device")
        if (handover.buf.dtype != torch.uint8 or not handover.buf.is_contiguous()
                or handover.buf.numel() < _size(_capi.selective_scan_handover_bytes, a.desc, *sizes)):
            raise ValueError("handover is not a buffer that the forward of this call filled")
        a.handover = handover.buf.data_ptr()
    a.workspace, a.workspace_bytes = _workspace(_size(_capi.selective_scan_bwd_workspace_bytes, a, *sizes, handed), dev, keep)
    _capi.selective_scan_bwd(a)
    return g


class SelectiveScanStep(_Step):
    """Streaming form of ``selective_scan_forward`` over preallocated buffers, ``GatedDeltaStep``'s counterpart: ``u``,
    ``dt``, ``z`` and ``out`` [B, T, D], ``B`` and ``C`` [B, T, N] or [B, T, G, N] hold the step's T new tokens (usually 1),
    ``state`` [B, D, N] is the contiguous float32 state, ``A``, ``D`` and ``dt_bias`` are contiguous float32. ``step()`` writes
    ``out`` and moves ``state`` on. It allocates nothing and does not synchronise, so a CUDA graph can capture it; refill the
    buffers in place between steps."""

    _run = "subq_selective_scan_fwd"

    def __init__(self, u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, out: torch.Tensor,
                 state: torch.Tensor, *, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                 dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = True, mask: Optional[torch.Tensor] = None):
        _require_cuda(u, dt, A, B, C, out, state)
        G = _scan_inputs(u, dt, A, B, C, z)
        _step_inner(u, dt, B, C, out, z)
        _step_mask(mask)
        N = A.shape[1]
        _own_buffer(A, "A", (u.shape[2], N), u.device)
        _own_buffer(D, "D", (u.shape[2],), u.device)
        _own_buffer(dt_bias, "dt_bias", (u.shape[2],), u.device)
        _check_out(out, u)
        keep: list = [u, dt, A, B, C, out, state, D, z, dt_bias, mask]
        with torch.cuda.device(u.device):
            a = _capi.SelectiveFwdArgs()
            a.desc = _scan_desc(u, A, D, dt_bias, dt_softplus, mask, G, keep)
            a.u, a.dt, a.z, a.B, a.C, a.out = _t3(u), _t3(dt), _t3(z), _t3(B), _t3(C), _t3(out)
            a.state_in = a.state_out = _own_buffer(state, "state", (u.shape[0], u.shape[2], N), u.device)
            a.workspace, a.workspace_bytes = _workspace(_capi.selective_scan_fwd_workspace_bytes(a), u.device, keep)
        self._set(a, u.device, keep)


# ---------------------------------------------------------------- residual RMSNorm
def _flat(t: torch.Tensor, keep: list) -> Tuple[int, int]:
    """(address, row stride) of t as [rows, D]: t itself where the leading dimensions merge, else a copy."""
    D = t.shape[-1]
    if not t.is_contiguous():
        t = t.reshape(-1, D)
        if D > 1 and t.stride(-1) != 1:
            t = t.contiguous()
        keep.append(t)
        return t.data_ptr(), t.stride(0)
    return t.data_ptr(), D


def _norm_types(x: torch.Tensor, residual: Optional[torch.Tensor]) -> torch.dtype:
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise ValueError("the norm needs a last dimension of 1 to 16384")
    if x.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {x.dtype}; use float32, float16 or bfloat16")
    if residual is None:
        return x.dtype
    if residual.shape != x.shape or residual.device != x.device:
        raise ValueError(f"residual must have x's shape {tuple(x.shape)} and device")
    if residual.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"residual must have x's type {x.dtype} or be float32, got {residual.dtype}")
    return residual.dtype


def _norm_run(x, weight, eps: float, residual, r_type, y_dtype: int, y: torch.Tensor, y_stride: int, scale: Optional[torch.Tensor], norm: int = 1
              ) -> Optional[torch.Tensor]:
    D, keep, r, res, rp = x.shape[-1], [], None, (None, 0), None
    if residual is not None:
        res = _flat(residual, keep)
        r = torch.empty(x.shape, dtype=r_type, device=x.device)
        rp = r.data_ptr()
    xp, xs = _flat(x, keep)
    _capi.rms_norm_fwd(_capi.RmsNormArgs(
        x.numel() // D, D, _DTYPES[x.dtype], _DTYPES[r_type], y_dtype, eps, norm, xp, xs, *res, rp, D, y.data_ptr(), y_stride,
        None if scale is None else scale.data_ptr(), 0 if scale is None else scale.shape[-1], _param(weight, "weight", (D,), x.device, keep),
        None, 0, None, 0, None, 0, None, 0, None, None, 0, _stream(x.device)))
    return r


@_on_its_device
def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5, *, residual: Optional[torch.Tensor] = None,
             out_dtype: Optional[torch.dtype] = None):
    """RMSNorm over the last dimension (1 to 16384 wide), with a residual's addition before it: r = x + residual, rounded to
    the residual's type (x's, or float32), y = r rsqrt(mean(r^2) + eps) weight. Returns ``y``, or ``(y, r)`` with a residual.
    ``out_dtype``: x's type, or float16 / bfloat16 for a float32 x. Math in float32; y and r are contiguous."""
    r_type = _norm_types(x, residual)
    y_type = x.dtype if out_dtype is None else out_dtype
    if y_type != x.dtype and not (x.dtype == torch.float32 and y_type in _TYPES):
        raise TypeError(f"the norm takes {x.dtype} into its own type (and float32 into a 16-bit type), not into {y_type}")
    y = torch.empty(x.shape, dtype=y_type, device=x.device)
    r = _norm_run(x, weight, eps, residual, r_type, _DTYPES[y_type], y, x.shape[-1], None)
    return y if residual is None else (y, r)


def _fp8_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Empty e4m3 rows of x's shape that start on 16-byte boundaries (what ``scaled_matmul`` reads as it is), and their scales."""
    *lead, D = x.shape
    q = torch.empty((*lead, (D + 15) // 16 * 16), dtype=_E4M3, device=x.device)
    return q[..., :D] if D % 16 else q, torch.empty((*lead, (D + _BLOCK - 1) // _BLOCK), dtype=torch.float32, device=x.device)


@_on_its_device
def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5, *, residual: Optional[torch.Tensor] = None):
    """``rms_norm`` with an 8-bit output: ``(q, scale)``, or ``(q, scale, r)`` with a residual. Every 128 columns of a row have
    a float32 scale = max(amax |y|, 1e-30) / 448 in ``scale`` [..., ceil(D / 128)], and ``q`` (float8_e4m3fn) is y / scale
    rounded to the nearest: what ``scaled_matmul`` multiplies with."""
    r_type = _norm_types(x, residual)
    q, scale = _fp8_rows(x)
    r = _norm_run(x, weight, eps, residual, r_type, _capi.SUBQ_E4M3, q, (x.shape[-1] + 15) // 16 * 16, scale)
    return (q, scale) if residual is None else (q, scale, r)


@_on_its_device
def quantize_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x in 8 bits, ``(q, scale)`` as ``rms_norm_fp8`` gives them, without a norm (a projection's input)."""
    _norm_types(x, None)
    q, scale = _fp8_rows(x)
    _norm_run(x, None, 0.0, None, x.dtype, _capi.SUBQ_E4M3, q, (x.shape[-1] + 15) // 16 * 16, scale, norm=0)
    return q, scale


@_on_its_device
def rms_norm_backward(dy: torch.Tensor, r: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
                      dresidual: Optional[torch.Tensor] = None, need_dweight: bool = True
                      ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of ``rms_norm`` from ``r`` (x itself, where there was no residual): ``(dx, dres, dweight | None)``.
    ``dresidual`` is the gradient that reaches r from elsewhere (the residual stream), of r's type; dx has dy's type (x's; of
    a float32 x normalised into 16 bits give dy in float32), dres has r's, and they are one tensor where the types are one.
    dweight is float32 [D], bitwise reproducible."""
    keep: list = []
    if dy.shape != r.shape or dy.device != r.device:
        raise ValueError("rms_norm_backward needs dy and r of one shape on one device")
    r_type, D = _norm_types(dy, r), r.shape[-1]
    (rp, rs), (gp, gs), (np_, ns) = _flat(r, keep), _flat(dy, keep), (None, 0)
    if dresidual is not None:
        if dresidual.shape != r.shape or dresidual.device != r.device or dresidual.dtype != r_type:
            raise ValueError("dresidual must have r's shape, type and device")
        np_, ns = _flat(dresidual, keep)
    dres = torch.empty(r.shape, dtype=r_type, device=r.device)
    dx = dres if dy.dtype == r_type else torch.empty(r.shape, dtype=dy.dtype, device=r.device)
    dw = torch.empty(D, dtype=torch.float32, device=r.device) if need_dweight else None
    a = _capi.RmsNormArgs(
        r.numel() // D, D, _DTYPES[dy.dtype], _DTYPES[r_type], _DTYPES[dy.dtype], eps, 1, None, 0, None, 0, rp, rs, None, 0, None, 0,
        _param(weight, "weight", (D,), r.device, keep), gp, gs, np_, ns, None if dx is dres else dx.data_ptr(), D, dres.data_ptr(), D,
        None if dw is None else dw.data_ptr(), None, 0, _stream(r.device))
    if dw is not None:
        a.workspace, a.workspace_bytes = _workspace(_size(_capi.rms_norm_bwd_workspace_bytes, a, D, a.rows > 0), r.device, keep)
    _capi.rms_norm_bwd(a)
    return dx, dres, dw


# --------------------------------------------------------------- 8-bit projection
def quantize_fp8_weight(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """A linear layer's weight [N, K] in 8 bits, ``(q, scale)``: a float32 scale = max(amax, 1e-30) / 448 for every 128 x 128 of
    it. For weights that are laid out once (torch operations, not a kernel)."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("quantize_fp8_weight takes a floating-point [N, K] weight")
    N, K = weight.shape
    n, k = (N + _BLOCK - 1) // _BLOCK, (K + _BLOCK - 1) // _BLOCK
    full = torch.zeros(n * _BLOCK, k * _BLOCK, dtype=torch.float32, device=weight.device)
    full[:N, :K] = weight.detach()
    blocks = full.view(n, _BLOCK, k, _BLOCK)
    scale = blocks.abs().amax((1, 3)).clamp_min(1e-30) / 448.0
    # (clamped: a quotient that is rounded up past 448 would be a NaN; a NaN weight stays one)
    q = (blocks / scale[:, None, :, None]).clamp(-448.0, 448.0).view(n * _BLOCK, k * _BLOCK)[:N, :(K + 15) // 16 * 16]
    return q.contiguous().to(_E4M3)[:, :K], scale


def _fp8_matrix(t: torch.Tensor, keep: list) -> Tuple[int, int]:
    """(address, row stride) of t as [rows, K], rows on 16-byte boundaries: t itself where it has them, else a copy."""
    K = t.shape[-1]
    if K % 16 == 0 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t.data_ptr(), K
    if t.dim() != 2:
        t = t.reshape(-1, K)
        keep.append(t)
    if (K > 1 and t.stride(1) != 1) or t.stride(0) % 16 or t.stride(0) < K or t.data_ptr() % 16:
        full = torch.empty(t.shape[0], (K + 15) // 16 * 16, dtype=t.dtype, device=t.device)
        full[:, :K].copy_(t)
        t = full
        keep.append(t)
    return t.data_ptr(), t.stride(0)


@_on_its_device
def scaled_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                  out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The projection of an 8-bit input with 8-bit weights: out = a b^T + bias, a [..., K] and b [N, K] float8_e4m3fn with float32
    scales, ``a_scale`` [..., ceil(K / 128)] for every 1 x 128 of a (``rms_norm_fp8``, ``quantize_fp8``) and ``b_scale``
    [ceil(N / 128), ceil(K / 128)] for every 128 x 128 of b (``quantize_fp8_weight``). Sums in float32; out [..., N] is
    float32, float16 or bfloat16. Rows that do not start on 16-byte boundaries are copied first (the quantising calls
    give rows that do). ``out`` is contiguous in its last dimension and shares no memory with the inputs."""
    if a.dtype is not _E4M3 or b.dtype is not _E4M3:
        raise TypeError(f"scaled_matmul takes float8_e4m3fn operands, got {a.dtype} and {b.dtype}")
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    *lead, K = a.shape
    if b.dim() != 2 or K != b.shape[1]:
        raise ValueError(f"shape mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}")
    N, nk = b.shape[0], (K + _BLOCK - 1) // _BLOCK
    if a_scale.shape != (*lead, nk) or b_scale.shape != ((N + _BLOCK - 1) // _BLOCK, nk):
        raise ValueError(f"a_scale must be {(*lead, nk)} and b_scale {((N + _BLOCK - 1) // _BLOCK, nk)}, got {tuple(a_scale.shape)} and {tuple(b_scale.shape)}")
    if a_scale.dtype is not torch.float32 or b_scale.dtype is not torch.float32:
        raise TypeError("scales must be float32")
    dev = a.device
    if not a.get_device() == b.get_device() == a_scale.get_device() == b_scale.get_device():
        _require_cuda(b, a_scale, b_scale)
        raise ValueError("the operands and their scales must be on one device")
    keep: list = []
    M = lead[0] if len(lead) == 1 else math.prod(lead)
    if out is None:
        out = torch.empty((*lead, N), dtype=out_dtype, device=dev)
        out_stride = N
    else:
        if out.shape != (*lead, N) or out.dtype != out_dtype or out.device != dev:
            raise ValueError(f"out must be {(*lead, N)} of {out_dtype} on the device of a")
        flat = out.view(-1, N) if N else out
        if N > 1 and flat.stride(-1) != 1:
            raise ValueError("out must have a contiguous last dimension")
        out_stride = flat.stride(0) if M > 1 else N
    if M and N:
        ap, a_s, bp, b_s, sap, sa_s, sbp, sb_s = None, 0, None, 0, None, 0, None, 0
        if K:
            (ap, a_s), (bp, b_s) = _fp8_matrix(a, keep), _fp8_matrix(b, keep)
            (sap, sa_s), (sbp, sb_s) = _flat(a_scale, keep), _flat(b_scale, keep)
        _capi.scaled_matmul(_capi.ScaledMatmulArgs(M, N, K, _DTYPES[out_dtype], ap, a_s, sap, sa_s, bp, b_s, sbp, sb_s, _param(bias, "bias", (N,), dev, keep),
                                                   out.data_ptr(), out_stride, _stream(dev)))
    return out
