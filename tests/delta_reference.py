"""The gated delta rule in float64, token by token, for the tests:

  S_t = gamma_t S_{t-1} + beta_t k_t (v_t - gamma_t S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t

differentiable by autograd (masked tokens leave S as it is and give o = 0)."""
import torch


def rule(q, k, v, beta, lg, mask, scale, S):
    """q, k, v [B, heads, N, *] (heads a divisor of H), beta, lg [B, H, N], S [B, H, d, e]: (o, S)."""
    B, H, N = beta.shape
    q, k, v = (x.repeat_interleave(H // x.shape[1], 1) for x in (q, k, v))
    out = []
    for t in range(N):
        D = lg[:, :, t, None, None].exp() * S
        w = v[:, :, t] - torch.einsum("bhde,bhd->bhe", D, k[:, :, t])
        new = D + beta[:, :, t, None, None] * k[:, :, t, :, None] * w[:, :, None, :]
        o = scale * torch.einsum("bhde,bhd->bhe", new, q[:, :, t])
        if mask is not None:
            m = mask[:, t].bool()[:, None, None]
            new, o = torch.where(m[..., None], new, S), torch.where(m, o, torch.zeros_like(o))
        S = new
        out.append(o)
    return (torch.stack(out, 2) if out else v.new_zeros(B, H, 0, v.shape[-1])), S


def clean(x, mask):
    """x [B, heads, N, ...] as float64 with 0 on masked tokens (whatever stood there)."""
    x = x.detach().double()
    if mask is None:
        return x
    m = mask.bool()[:, None, :] if x.dim() == 3 else mask.bool()[:, None, :, None]
    return torch.where(m, x, torch.zeros_like(x))


def forward(q, k, v, beta, lg, mask, scale, S0):
    B, _, N, d = q.shape
    H = beta.shape[1]
    S = torch.zeros(B, H, d, v.shape[-1], dtype=torch.float64, device=q.device) if S0 is None else S0.double()
    with torch.no_grad():
        return rule(*(clean(x, mask) for x in (q, k, v, beta, lg)), mask, scale, S)


def gradients(q, k, v, beta, lg, mask, scale, S0, do, dS):
    """(dq, dk, dv, dbeta, dlg, dS0) in float64."""
    B, _, N, d = q.shape
    H = beta.shape[1]
    S = torch.zeros(B, H, d, v.shape[-1], dtype=torch.float64, device=q.device) if S0 is None else S0.double()
    leaves = [clean(x, mask).requires_grad_(True) for x in (q, k, v, beta, lg)] + [S.clone().requires_grad_(True)]
    o, S_end = rule(*leaves[:5], mask, scale, leaves[5])
    loss = (o * clean(do, mask)).sum()
    if dS is not None:
        loss = loss + (S_end * dS.double()).sum()
    got = torch.autograd.grad(loss, leaves, allow_unused=True)
    return [torch.zeros_like(x) if g is None else g for g, x in zip(got, leaves)]
