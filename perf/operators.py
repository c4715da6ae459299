"""Cases of the gated delta rule and of layer norm: what a pass of each is, on which inputs, and what it has to compute.

Two families of operators:

* the gated delta rule over [B, H, N, d] heads: for each (batch, head) a state S [d, e] that every live token decays and corrects,

      S_t = gamma_t S_{t-1} + beta_t k_t (v_t - gamma_t S_{t-1}^T k_t)^T,      o_t = scale S_t^T q_t,

  over a whole prompt (``prefill``), with its gradients (``train``), and for one new token a sequence (``decode``);
* layer norm over the last dimension (``ln``), and with its gradients (``ln_train``).

``own`` False: plain forms in elementary torch operations, float32 inside, rounded once at the end. ``own`` True: the calls a user
makes of this repository's operators. ``exact`` gives the same outputs from the definitions in float64.
"""
import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sub-quadratic-audio-transformer-engine_b200")
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _ops():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from subq_audio import ops

    return ops


# ---------------------------------------------------------------------------------------------------------------- the cases
def _delta(name, kind, B, H, Hq, Hkv, N, d, e, dtype, state=False, ragged=False):
    """H heads of beta, gamma and the state; q has Hq heads and k, v have Hkv (divisors of H)."""
    case = {"kind": kind, "B": B, "H": H, "Hq": Hq, "Hkv": Hkv, "N": N, "d": d, "e": e, "dtype": dtype, "state": state, "ragged": ragged}
    return dict(case, name=name) if name else case


def _norm(name, kind, rows, dim, x, y):
    case = {"kind": kind, "rows": rows, "dim": dim, "x": x, "y": y}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one piece of a long audio stream: 4 heads, 4096 new tokens from a carried state, the state handed on
        _delta("prefill stream piece", "prefill", 1, 4, 4, 4, 4096, 64, 64, "fp16", state=True),
        # a padded batch of prompts of different, odd lengths; the states start a generation
        _delta("prefill ragged batch", "prefill", 8, 12, 12, 12, 2047, 64, 64, "bf16", state=True, ragged=True),
        # one very long recording: few sequences, so the work has to be split over time
        _delta("prefill long", "prefill", 1, 12, 12, 12, 65536, 64, 64, "bf16", state=True),
        # wide heads, four of them sharing a key and value head
        _delta("prefill wide grouped", "prefill", 2, 16, 16, 4, 4096, 128, 128, "bf16"),
        # the training step of the default benchmark's shape, with padding
        _delta("train batch", "train", 8, 8, 8, 8, 8192, 64, 64, "bf16", ragged=True),
        # a float32 fine-tuning step with grouped keys and values and an odd length
        _delta("train grouped fp32", "train", 2, 12, 12, 4, 1537, 64, 64, "fp32"),
        # one stream's next token: latency is all there is
        _delta("decode one", "decode", 1, 12, 12, 12, 1, 64, 64, "bf16", state=True),
        # a server's next tokens: the states' bytes
        _delta("decode batch", "decode", 256, 12, 12, 12, 1, 64, 64, "bf16", state=True),
        # the norm before a layer for one new token
        _norm("layer norm one row", "ln", 1, 768, "fp32", "bf16"),
        # the norm before a layer of the encoder's batch: the float32 residual in, the projections' bf16 input out
        _norm("layer norm encoder", "ln", 65536, 768, "fp32", "bf16"),
        # its training step
        _norm("layer norm train encoder", "ln_train", 65536, 768, "fp32", "bf16"),
        # an odd width and an odd number of rows, all in bf16
        _norm("layer norm train odd", "ln_train", 4999, 1021, "bf16", "bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "train", "train", "decode", "ln", "ln_train"])
    if kind in ("ln", "ln_train"):
        dim = rng.choice([256, 384, 512, 768, 1024, 1280, _log(rng, 8, 8192) | 1, _log(rng, 64, 8192)])
        x, y = rng.choice([("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32"), ("fp32", "fp16")])
        return _norm(None, kind, _log(rng, 1, max(1, 48_000_000 // dim)), dim, x, y)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    d, e = rng.choice([(64, 64), (64, 64), (128, 128), (32, 32), (64, 128), (128, 64), (80, 80), (48, 96)])
    G = rng.choice([1, 1, 2, 4])
    Hkv = rng.choice([1, 2, 3, 4])
    H = Hkv * G
    if kind == "decode":
        B = _log(rng, 1, max(1, 256 * 12 * 64 * 64 // (H * d * e)))
        return _delta(None, kind, B, H, H, Hkv, 1, d, e, dtype, state=True)
    most = {"prefill": 700_000, "train": 400_000}[kind] * 64 * 64 // max(d * e, 64 * 64) * 2 // _SIZE[dtype]
    N = _log(rng, 17, min(16384, most // H))
    B = _log(rng, 1, max(1, min(16, most // (H * N))))
    return _delta(None, kind, B, H, H, Hkv, N, d, e, dtype, state=kind == "prefill" and rng.random() < 0.5, ragged=rng.random() < 0.4 and N > 8)


def _lens(case):
    """Live tokens of each row of a ragged batch: from half the length to all of it."""
    B, N = case["B"], case["N"]
    return [N if not case["ragged"] or B == 1 and N < 2 else N - (N // 2) * i // max(1, B) for i in range(B)]


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["kind"] in ("ln", "ln_train"):
        rows, dim = case["rows"], case["dim"]
        # a residual stream: channels of different scales and offsets
        x = randn(rows, dim) * (0.5 + randn(dim).abs()) + 0.3 * randn(dim)
        s = {"x": x.to(_TYPES[case["x"]]), "weight": 1 + 0.2 * randn(dim), "bias": 0.1 * randn(dim)}
        if case["kind"] == "ln_train":
            s["dy"] = randn(rows, dim).to(_TYPES[case["y"]])
        return s
    B, H, Hq, Hkv, N, d, e = (case[n] for n in ("B", "H", "Hq", "Hkv", "N", "d", "e"))
    t = _TYPES[case["dtype"]]

    def heads(h, w, unit):  # a [B, h, N, w] view of a projection's [B, N, h, w] output
        x = randn(B, N, h, w)
        if unit:  # queries and keys come normalised
            x = x / x.square().sum(-1, keepdim=True).sqrt()
        return x.to(t).transpose(1, 2)

    s = {"q": heads(Hq, d, True), "k": heads(Hkv, d, True), "v": heads(Hkv, e, False)}
    s["beta"] = torch.sigmoid(randn(B, N, H)).transpose(1, 2)
    # gates from about 0.5 to 1, each head with a mean of its own, as a gate projection gives them
    s["log_gamma"] = -torch.nn.functional.softplus(-(randn(B, N, H) + 1 + 4 * torch.rand(H, generator=g, device="cuda"))).transpose(1, 2)
    s["mask"] = None
    if case["ragged"]:
        lens = torch.tensor(_lens(case), device="cuda")[torch.randperm(B, generator=g, device="cuda")]
        s["mask"] = torch.arange(N, device="cuda")[None, :] < lens[:, None]
    s["state"] = 0.5 * randn(B, H, d, e) if case["state"] else None
    if case["kind"] == "train":
        s["dout"] = randn(B, N, H, e).to(t).transpose(1, 2)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["kind"] = case["kind"]
    s["out_dtype"] = _TYPES[case["y"]] if "y" in case else None
    if case["kind"] == "decode":
        # a serving loop's buffers, refilled between steps, and its handle on them
        s["beta"], s["log_gamma"] = s["beta"].contiguous(), s["log_gamma"].contiguous()
        s["out"] = torch.empty(case["B"], case["H"], 1, case["e"], device="cuda", dtype=s["q"].dtype)
        if own:
            s["step"] = _ops().GatedDeltaStep(s["q"], s["k"], s["v"], s["beta"], s["out"], s["state"], log_gamma=s["log_gamma"])
    return s


# ---------------------------------------------------------------------------------------------------------------- the plain forms
_CHUNK = 64


def _unit_lower_inverse(A):
    """(I + A)^-1 of strictly lower triangular [..., C, C] matrices, by doubling the size of the inverted diagonal blocks."""
    C = A.shape[-1]
    lead = A.shape[:-2]
    T = torch.ones(*lead, C, 1, 1, dtype=A.dtype, device=A.device)
    s = 1
    while s < C:
        n = C // (2 * s)
        low = A.reshape(*lead, n, 2, s, n, 2, s)[..., :, 1, :, :, 0, :].diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        T = T.reshape(*lead, n, 2, s, s)
        a, b = T[..., 0, :, :], T[..., 1, :, :]
        T = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([-(b @ low @ a), b], -1)], -2)
        s *= 2
    return T.reshape(*lead, C, C)


def _plain_delta(q, k, v, beta, lg, mask, scale, S):
    """Float32 chunked form: within a chunk the corrections solve a triangular system, between chunks the state is carried."""
    B, H, N = beta.shape
    d, e = q.shape[-1], v.shape[-1]
    q, k, v = (x.repeat_interleave(H // x.shape[1], 1) for x in (q, k, v))
    if mask is not None:
        live = mask[:, None, :, None]
        q, k, v = (torch.where(live, x, torch.zeros_like(x)) for x in (q, k, v))
        beta, lg = (torch.where(mask[:, None, :], x, torch.zeros_like(x)) for x in (beta, lg))
    pad = -N % _CHUNK
    n = (N + pad) // _CHUNK
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)).reshape(B, H, n, _CHUNK, -1) for x in (q, k, v))
    beta, lg = (torch.nn.functional.pad(x, (0, pad)).reshape(B, H, n, _CHUNK) for x in (beta, lg))
    g = lg.cumsum(-1)
    lower = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device).tril()
    gamma = torch.where(lower, g[..., :, None] - g[..., None, :], torch.full_like(g[..., None], -math.inf)).exp()
    A = (beta[..., None] * (k @ k.mT) * gamma).tril(-1)
    P = (q @ k.mT) * gamma
    T = _unit_lower_inverse(A)
    eg = g.exp()[..., None]
    U = T @ (beta[..., None] * v)
    W = T @ (beta[..., None] * eg * k)
    qg = q * eg
    kg = k * (g[..., -1:] - g).exp()[..., None]
    last = eg[..., -1:, :]
    if S is None:
        S = torch.zeros(B, H, d, e, device=q.device)
    out = []
    for c in range(n):
        u = U[:, :, c] - W[:, :, c] @ S
        out.append(qg[:, :, c] @ S + P[:, :, c] @ u)
        S = last[:, :, c] * S + kg[:, :, c].mT @ u
    return (scale * torch.stack(out, 2)).reshape(B, H, n * _CHUNK, e)[:, :, :N], S


def _plain_step(s):
    H = s["beta"].shape[1]
    q, k, v = (s[n].float().repeat_interleave(H // s[n].shape[1], 1) for n in ("q", "k", "v"))
    S = s["log_gamma"].exp()[..., None] * s["state"]
    u = s["beta"][..., None] * (v - k @ S)
    S = S + k.mT @ u
    s["state"].copy_(S)
    s["out"].copy_(q.shape[-1] ** -0.5 * (q @ S))
    return s["out"], s["state"]


def _plain_norm(s):
    x = s["x"].float()
    xc = x - x.mean(-1, keepdim=True)
    r = (xc.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xh = xc * r
    y = (xh * s["weight"] + s["bias"]).to(s["out_dtype"])
    if s["kind"] == "ln":
        return y
    dy = s["dy"].float()
    gw = dy * s["weight"]
    dx = r * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xh).sum(0), dy.sum(0)


def _run_plain(s):
    if s["kind"] in ("ln", "ln_train"):
        return _plain_norm(s)
    if s["kind"] == "decode":
        return _plain_step(s)
    t = s["q"].dtype
    scale = s["q"].shape[-1] ** -0.5
    if s["kind"] == "prefill":
        o, S = _plain_delta(s["q"].float(), s["k"].float(), s["v"].float(), s["beta"], s["log_gamma"], s["mask"], scale, s["state"])
        return (o.to(t), S) if s["state"] is not None else o.to(t)
    leaves = [s[n].detach().float().requires_grad_(True) for n in ("q", "k", "v", "beta", "log_gamma")]
    o, _ = _plain_delta(*leaves, s["mask"], scale, None)
    dq, dk, dv, dbeta, dlg = torch.autograd.grad(o, leaves, s["dout"].float())
    return o.detach().to(t), dq.to(t), dk.to(t), dv.to(t), dbeta, dlg


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    ops = _ops()
    if s["kind"] in ("ln", "ln_train"):
        y = ops.layer_norm(s["x"], s["weight"], s["bias"], 1e-5, out_dtype=s["out_dtype"])
        if s["kind"] == "ln":
            return y
        return (y,) + tuple(ops.layer_norm_backward(s["dy"], s["x"], s["weight"], 1e-5))
    if s["kind"] == "decode":
        s["step"].step()
        return s["out"], s["state"]
    if s["kind"] == "prefill":
        o, S = ops.gated_delta_forward(s["q"], s["k"], s["v"], s["beta"], log_gamma=s["log_gamma"], mask=s["mask"], state=s["state"],
                                       return_state=s["state"] is not None)
        return (o, S) if s["state"] is not None else o
    handover = ops.DeltaHandover()
    o, _ = ops.gated_delta_forward(s["q"], s["k"], s["v"], s["beta"], log_gamma=s["log_gamma"], mask=s["mask"], handover=handover)
    dq, dk, dv, dbeta, dlg, _ = ops.gated_delta_backward(s["q"], s["k"], s["v"], s["beta"], s["dout"], log_gamma=s["log_gamma"],
                                                         mask=s["mask"], need_dlog_gamma=True, handover=handover)
    return o, dq, dk, dv, dbeta, dlg


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------- the work
def work(case):
    if case["kind"] in ("ln", "ln_train"):
        n = case["rows"] * case["dim"]
        x, y = _SIZE[case["x"]], _SIZE[case["y"]]
        if case["kind"] == "ln":
            return {"bytes": n * (x + y) + 8 * case["dim"], "flops": 8 * n}
        # x once for both passes is not possible between two calls: x and y of the forward, x, dy and dx of the backward
        return {"bytes": n * (x + y + x + y + x) + 20 * case["dim"], "flops": 24 * n}
    B, H, Hq, Hkv, N, d, e = (case[n] for n in ("B", "H", "Hq", "Hkv", "N", "d", "e"))
    live = sum(_lens(case))
    t = _SIZE[case["dtype"]]
    into = live * (Hq * d + Hkv * (d + e)) * t + live * H * 8  # q, k, v, beta, log gamma of the live tokens
    out = B * N * H * e * t
    states = 2 * B * H * d * e * 4 if case["state"] else 0
    flops = 6 * live * H * d * e  # S^T k, the rank-one correction, S^T q
    mask = B * N if case["ragged"] else 0
    if case["kind"] != "train":
        return {"bytes": into + out + states + mask, "flops": flops}
    grads = B * N * (Hq * d + Hkv * (d + e)) * t + B * N * H * 8
    return {"bytes": 2 * into + out + live * H * e * t + grads + mask, "flops": 3 * flops}


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_delta(s, dout):
    """Token by token; the gradients from the adjoint recurrence, with the states recomputed from every 64th."""
    H = s["beta"].shape[1]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    groups = [H // x.shape[1] for x in (q, k, v)]
    q, k, v = (x[:, torch.arange(H, device=x.device) // n] for x, n in zip((q, k, v), groups))
    B, _, N, d = q.shape
    e = v.shape[-1]
    live = torch.ones(B, N, dtype=torch.bool, device=q.device) if s["mask"] is None else s["mask"]
    m = live[:, None, :].double()
    beta, gamma = s["beta"].double() * m, torch.exp(s["log_gamma"].double() * m)
    scale = d ** -0.5
    S = torch.zeros(B, H, d, e, dtype=torch.float64, device=q.device) if s["state"] is None else s["state"].double()

    def step(S, t):  # (decayed state, correction, new state)
        D = gamma[:, :, t, None, None] * S
        w = v[:, :, t] - torch.einsum("bhde,bhd->bhe", D, k[:, :, t])
        return D, w, D + k[:, :, t, :, None] * (beta[:, :, t, None] * w)[:, :, None, :]

    o = torch.zeros(B, H, N, e, dtype=torch.float64, device=q.device)
    marks = []
    for t in range(N):
        if t % 64 == 0:
            marks.append(S)
        S = step(S, t)[2]
        o[:, :, t] = scale * torch.einsum("bhde,bhd->bhe", S, q[:, :, t])
    o = o * m[..., None]
    if dout is None:
        return o, S
    do = dout.double() * m[..., None]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dbeta, dlg = torch.zeros_like(beta), torch.zeros_like(beta)
    G = torch.zeros_like(S)
    for c in reversed(range(len(marks))):
        S, kept = marks[c], []
        for t in range(64 * c, min(N, 64 * c + 64)):
            D, w, S = step(S, t)
            kept.append((t, D, w, S))
        for t, D, w, S_t in reversed(kept):
            kt, b = k[:, :, t], beta[:, :, t]
            G = G + scale * q[:, :, t, :, None] * do[:, :, t, None, :]
            dq[:, :, t] = scale * torch.einsum("bhde,bhe->bhd", S_t, do[:, :, t])
            r = torch.einsum("bhde,bhd->bhe", G, kt)
            br = b[..., None] * r
            dv[:, :, t] = br
            dbeta[:, :, t] = (r * w).sum(-1)
            dk[:, :, t] = torch.einsum("bhde,bhe->bhd", G, b[..., None] * w) - torch.einsum("bhde,bhe->bhd", D, br)
            G = G - kt[..., None] * br[:, :, None, :]
            dlg[:, :, t] = (G * D).sum((-1, -2))
            G = gamma[:, :, t, None, None] * G
    dq, dk, dv = (x * m[..., None] for x in (dq, dk, dv))
    dq, dk, dv = (x.reshape(B, H // n, n, N, -1).sum(2) for x, n in zip((dq, dk, dv), groups))
    return o, dq, dk, dv, dbeta * m, dlg * m


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("ln", "ln_train"):
        if case["rows"] * case["dim"] > 100_000_000:
            return None
        x, w = s["x"].double(), s["weight"].double()
        mean = x.sum(-1) / case["dim"]
        sd = ((x - mean[:, None]).pow(2).sum(-1) / case["dim"] + 1e-5).sqrt()
        z = (x - mean[:, None]) / sd[:, None]
        y = z * w + s["bias"].double()
        if case["kind"] == "ln":
            return y
        dy = s["dy"].double()
        dz = dy * w
        dx = (dz - (dz.sum(-1)[:, None] + z * (dz * z).sum(-1)[:, None]) / case["dim"]) / sd[:, None]
        return y, dx, (dy * z).sum(0), dy.sum(0)
    if case["kind"] == "decode":
        H = case["H"]
        q, k, v = (s[n].double()[:, :, 0].repeat_interleave(H // s[n].shape[1], 1) for n in ("q", "k", "v"))
        D = s["log_gamma"].double().exp()[..., None] * s["state"].double()
        S = D + s["beta"].double()[..., None] * k[..., None] * (v - (D * k[..., None]).sum(-2))[:, :, None, :]
        return (case["d"] ** -0.5 * (S * q[..., None]).sum(-2))[:, :, None], S
    got = _exact_delta(s, s.get("dout"))
    return got if case["kind"] == "train" or case["state"] else got[0]
