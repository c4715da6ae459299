"""Definitions in float64 of a selective state space block's operators, token by token, differentiable by torch's autograd."""
import torch


def softplus(x):
    return x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))


def silu(x):
    return x * torch.sigmoid(x)


def scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, mask=None, state=None):
    """[B, L, D] inputs, B and C [B, L, G, N]; all float64. Returns (out, state)."""
    Bn, L, Dn = u.shape
    group = torch.arange(Dn, device=u.device) // (Dn // B.shape[2])
    h = torch.zeros(Bn, Dn, A.shape[1], dtype=u.dtype, device=u.device) if state is None else state
    out = []
    for t in range(L):
        step = dt[:, t] if dt_bias is None else dt[:, t] + dt_bias
        step = softplus(step) if dt_softplus else step
        new = torch.exp(step[..., None] * A) * h + (step * u[:, t])[..., None] * B[:, t, group]
        y = (new * C[:, t, group]).sum(-1)
        if D is not None:
            y = y + D * u[:, t]
        if z is not None:
            y = y * silu(z[:, t])
        if mask is not None:
            live = mask[:, t, None]
            new, y = torch.where(live[..., None], new, h), torch.where(live, y, torch.zeros_like(y))
        h = new
        out.append(y)
    return (torch.stack(out, 1) if out else u * 0), h


def conv(x, w, b=None, activation="silu", mask=None, state=None):
    """Returns (y, window behind the last live token)."""
    Bn, L, D = x.shape
    W = w.shape[1]
    if mask is not None:
        x = torch.where(mask[..., None], x, torch.zeros_like(x))
    first = torch.zeros(Bn, W - 1, D, dtype=x.dtype, device=x.device) if state is None else state
    seen = torch.cat([first, x], 1)
    y = sum(w[:, j] * seen[:, j:j + L] for j in range(W))
    if b is not None:
        y = y + b
    if activation == "silu":
        y = silu(y)
    ends = [L] * Bn
    if mask is not None:
        y = torch.where(mask[..., None], y, torch.zeros_like(y))
        ends = [int(m.nonzero().max()) + 1 if bool(m.any()) else 0 for m in mask]
    return y, torch.stack([seen[i, e:e + W - 1] for i, e in enumerate(ends)]) if Bn else first


def to_e4m3(x):
    """Float64 values rounded to e4m3 (nearest, ties to even), as float64."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def quantize(y):
    """(q, scale) of float64 rows. y / (amax / 448) is formed as 448 y / amax, whose first product is exact: 16-bit values hit the
    middle between two e4m3 values exactly, which the rounding of amax / 448 would push to either side."""
    D = y.shape[-1]
    parts = [y[..., i:i + 128] for i in range(0, D, 128)]
    top = torch.stack([p.abs().amax(-1).clamp_min(1e-30) for p in parts], -1)
    return torch.cat([to_e4m3(448 * p / s[..., None]) for p, s in zip(parts, top.unbind(-1))], -1), top / 448


def rms(r, w=None, eps=1e-5):
    y = r / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    return y if w is None else y * w


def matmul(a, a_scale, b, b_scale, bias=None):
    K, N = a.shape[-1], b.shape[0]
    out = 0
    for i in range(a_scale.shape[-1]):
        k = slice(128 * i, min(K, 128 * i + 128))
        rows = b_scale[:, i].double().repeat_interleave(128)[:N]
        out = out + (a[..., k].double() @ b[:, k].double().t()) * a_scale[..., i, None].double() * rows
    return out if bias is None else out + bias.double()
