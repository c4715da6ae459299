"""The gated delta rule in float64 by chunks of tokens, for sequences too long to walk token by token:

  U = (I + A)^-1 (beta (V - e^g K S)),   A_ij = beta_i e^{g_i - g_j} k_i.k_j for i > j,
  O = scale (e^g Q S + tril(e^{g_i - g_j} q_i.k_j) U),   S' = e^{g_C} S + (e^{g_C - g} K)^T U

with g the running sum of log gamma in the chunk; differentiable by autograd. A masked token is one with
k = 0, beta = 0 and log gamma = 0 whose output is not used (test_delta_chunk_reference.py: equal to the
rule token by token)."""
import torch

from delta_reference import clean

CHUNK = 128


def rule(q, k, v, beta, lg, mask, scale, S):
    """q, k, v [B, heads, N, *] (heads a divisor of H), beta, lg [B, H, N], S [B, H, d, e], float64: (o, S)."""
    H, N = beta.shape[1:]
    q, k, v = (x.repeat_interleave(H // x.shape[1], 1) for x in (q, k, v))
    out = []
    for n in range(0, N, CHUNK):
        K, Q, V, be = (x[:, :, n:n + CHUNK] for x in (k, q, v, beta))
        g = lg[:, :, n:n + CHUNK].cumsum(-1)
        C = g.shape[-1]
        low = torch.ones(C, C, dtype=torch.bool, device=g.device).tril()
        G = (g[..., :, None] - g[..., None, :]).masked_fill(~low, 0.0).exp() * low
        eg = g.exp()[..., None]
        A = be[..., None] * (G * (K @ K.mT)).tril(-1)
        U = torch.linalg.solve_triangular(A + torch.eye(C, dtype=A.dtype, device=A.device), be[..., None] * (V - eg * (K @ S)),
                                          upper=False, unitriangular=True)
        O = scale * (eg * (Q @ S) + (G * (Q @ K.mT)) @ U)
        S = g[..., -1, None, None].exp() * S + ((g[..., -1:] - g).exp()[..., None] * K).mT @ U
        out.append(O if mask is None else torch.where(mask[:, None, n:n + CHUNK, None].bool(), O, torch.zeros_like(O)))
    return torch.cat(out, 2), S


def _leaves(q, k, v, beta, lg, mask, S0):
    B, H, _ = beta.shape
    S = torch.zeros(B, H, q.shape[-1], v.shape[-1], dtype=torch.float64, device=q.device) if S0 is None else S0.double()
    return [clean(x, mask) for x in (q, k, v, beta, lg)] + [S]


def forward(q, k, v, beta, lg, mask, scale, S0):
    *x, S = _leaves(q, k, v, beta, lg, mask, S0)
    with torch.no_grad():
        return rule(*x, mask, scale, S)


def gradients(q, k, v, beta, lg, mask, scale, S0, do, dS):
    """(dq, dk, dv, dbeta, dlg, dS0) in float64, 0 on masked tokens."""
    leaves = [x.clone().requires_grad_(True) for x in _leaves(q, k, v, beta, lg, mask, S0)]
    o, S = rule(*leaves[:5], mask, scale, leaves[5])
    loss = (o * clean(do, mask)).sum()
    if dS is not None:
        loss = loss + (S * dS.double()).sum()
    got = torch.autograd.grad(loss, leaves)
    return [clean(g, mask) for g in got[:5]] + [got[5]]
