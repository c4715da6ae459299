"""Inputs of the gated delta rule whose state lasts across segments of a sequence, and the rule by segments in float64.

Keys lean towards one direction after another (97 tokens each, the directions share a part), beta is 0.01 to 0.05 and the
decay absent or 1e-4 a token: what a segment does to the state before it, M, then erases some directions in an order, so
that M is neither 0, the identity nor symmetric."""
import torch

import delta_chunk_reference as ref

# (d, e, type, N, log gamma, masked)
CASES = [(48, 96, "bf16", 4096, -1e-4, False), (64, 64, "bf16", 4096, 0.0, True), (80, 40, "bf16", 3000, 0.0, False),
         (100, 64, "bf16", 3000, -1e-4, True), (128, 128, "bf16", 2950, 0.0, False),
         (48, 48, "fp16", 3333, 0.0, True), (64, 200, "fp16", 2500, -1e-4, False), (80, 80, "fp16", 2500, -1e-4, False),
         (100, 33, "fp16", 2500, 0.0, False), (128, 64, "fp16", 2500, -1e-4, True),
         (48, 64, "fp32", 2500, -1e-4, False), (64, 64, "fp32", 2500, 0.0, True), (80, 80, "fp32", 2500, 0.0, False),
         (100, 40, "fp32", 2500, -1e-4, True), (128, 128, "fp32", 2500, 0.0, False)]
IDS = ["-".join(str(x) for x in c) for c in CASES]
T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def inputs(d, e, dtype, N, lowest, masked, B=1, H=2, Hk=1):
    g = torch.Generator().manual_seed(N + 3 * d + e)

    def randn(*shape):
        return torch.randn(*shape, generator=g)

    def unit(x):
        return x / x.norm(dim=-1, keepdim=True)

    turns = (N + 96) // 97
    lean = unit(unit(randn(B, Hk, 1, d)) + unit(randn(B, Hk, turns, d))).repeat_interleave(97, 2)[:, :, :N]
    q, k = unit(randn(B, H, N, d)).to(T[dtype]), unit(lean + 0.5 * unit(randn(B, Hk, N, d))).to(T[dtype])
    v, do = (0.5 + randn(B, H, N, e)).to(T[dtype]), (0.5 + randn(B, H, N, e)).to(T[dtype])
    beta = 0.01 + 0.04 * torch.rand(B, H, N, generator=g)
    lg = lowest * torch.rand(B, H, N, generator=g)
    m = torch.rand(B, N, generator=g) < 0.8 if masked else None
    return q, k, v, do, beta, lg, 1 + randn(B, H, d, e), 1 + randn(B, H, d, e), m


def by_segments(q, k, v, beta, lg, mask, scale, S, length, transition=lambda M: M):
    """The rule with each segment's result on S as M S + L; `transition` stands in for M (an error to plant)."""
    q, k, v, beta, lg = (ref.clean(x, mask) for x in (q, k, v, beta, lg))
    H, N, d = beta.shape[1], beta.shape[2], q.shape[-1]
    out, S = [], S.double()
    for n in range(0, N, length):
        x = [t[:, :, n:n + length] for t in (q, k, v, beta, lg)]
        m = None if mask is None else mask[:, n:n + length]
        out.append(ref.rule(*x, m, scale, S)[0])
        eye = torch.eye(d, dtype=S.dtype, device=S.device).expand(S.shape[0], H, d, d)
        M = ref.rule(x[0], x[1], torch.zeros_like(x[0]), x[3], x[4], m, scale, eye)[1]
        L = ref.rule(*x, m, scale, torch.zeros_like(S))[1]
        S = (transition(M) if n else M) @ S + L
    return torch.cat(out, 2), S
