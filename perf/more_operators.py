"""Cases of a selective state space block's operators: what a pass of each is, on which inputs, and what it has to compute.

* the selective scan over [B, L, D] channels, each with N states (``scan``, with its gradients ``scan_train``):

      dt_t = softplus(raw_t + bias),   h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   y_t = (C_t . h_t + D u_t) silu(z_t);

* the short causal convolution before it (``conv``, ``conv_train``): y_t = silu(b + sum_j w_j x_{t-W+1+j}), one filter a channel;
* both for one new token a sequence (``step``), from the carried inputs and states, which are updated in place;
* the root-mean-square norm before the block, with the residual's addition (``norm_train``), or with an 8-bit output and a scale for
  every 128 of a row (``norm_fp8``);
* the projection of such an output with weights in 8 bits and a scale for every 128 x 128 of them (``matmul``).

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
_BLOCK = 128
_TOP = 448.0  # the largest e4m3 value


def _ops():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from subq_audio import ops

    return ops


# ---------------------------------------------------------------------------------------------------------------- the cases
def _scan(name, kind, B, L, D, N, G, dtype, gate=True, state=False, ragged=False):
    """D channels of N states; B and C are shared by D / G channels."""
    case = {"kind": kind, "B": B, "L": L, "D": D, "N": N, "G": G, "dtype": dtype, "gate": gate, "state": state, "ragged": ragged}
    return dict(case, name=name) if name else case


def _conv(name, kind, B, L, D, W, dtype, state=False, ragged=False):
    case = {"kind": kind, "B": B, "L": L, "D": D, "W": W, "dtype": dtype, "state": state, "ragged": ragged}
    return dict(case, name=name) if name else case


def _step(name, B, D, N, W, dtype):
    case = {"kind": "step", "B": B, "D": D, "N": N, "W": W, "G": 1, "L": 1, "dtype": dtype}
    return dict(case, name=name) if name else case


def _norm(name, kind, rows, dim, x, r):
    case = {"kind": kind, "rows": rows, "dim": dim, "x": x, "r": r}
    return dict(case, name=name) if name else case


def _matmul(name, M, N, K, dtype):
    case = {"kind": "matmul", "M": M, "N": N, "K": K, "dtype": dtype}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one piece of a long audio stream: 4096 new tokens behind the last inputs of the piece before
        _conv("conv stream piece", "conv", 1, 4096, 1536, 4, "fp16", state=True),
        # the training step of a padded batch
        _conv("conv train batch", "conv_train", 8, 2047, 1536, 4, "bf16", ragged=True),
        # a padded batch of prompts of different, odd lengths; the states start a generation
        _scan("scan ragged batch", "scan", 8, 2047, 1536, 16, 1, "bf16", state=True, ragged=True),
        # one very long recording: few channels, so the work has to be split over time
        _scan("scan long", "scan", 1, 65536, 1536, 16, 1, "bf16", state=True),
        # the training step of a batch
        _scan("scan train batch", "scan_train", 4, 2048, 1536, 16, 1, "bf16"),
        # a float32 fine-tuning step with an odd length and two groups of B and C, without a gate
        _scan("scan train grouped fp32", "scan_train", 2, 1537, 384, 16, 2, "fp32", gate=False),
        # one stream's next token: latency is all there is
        _step("step one", 1, 1536, 16, 4, "bf16"),
        # a server's next tokens: the states' bytes
        _step("step batch", 256, 1536, 16, 4, "bf16"),
        # the norm before the 8-bit projection of a batch of prompts
        _norm("norm to 8 bits prompts", "norm_fp8", 16384, 1024, "bf16", "bf16"),
        # the training step of the norm before a layer of the encoder: bf16 branch, float32 residual stream
        _norm("norm train encoder", "norm_train", 65536, 768, "bf16", "fp32"),
        # the projection into the block, of a batch of prompts
        _matmul("matmul prompts", 16384, 4096, 1024, "bf16"),
        # the same for one stream's next token: the weights' bytes
        _matmul("matmul one token", 1, 4096, 1024, "bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["conv", "conv_train", "scan", "scan", "scan_train", "scan_train", "step", "norm_fp8", "norm_train", "matmul", "matmul"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("norm_fp8", "norm_train"):
        dim = rng.choice([256, 512, 768, 1024, 2048, _log(rng, 8, 8192) | 1, _log(rng, 64, 8192)])
        x, r = rng.choice([("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
        return _norm(None, kind, _log(rng, 1, max(1, (16_000_000 if kind == "norm_fp8" else 48_000_000) // dim)), dim, x, r)
    if kind == "matmul":
        K = rng.choice([512, 768, 1024, 2048, _log(rng, 64, 4096), _log(rng, 64, 4096) | 1])
        N = rng.choice([768, 1024, 1536, 4096, _log(rng, 32, 8192), _log(rng, 32, 8192) | 1])
        return _matmul(None, _log(rng, 1, max(1, min(16384, 60_000_000_000 // (N * K)))), N, K, "bf16" if dtype == "bf16" else rng.choice(["fp16", "fp32"]))
    if kind in ("conv", "conv_train"):
        D = rng.choice([384, 768, 1024, 1536, _log(rng, 16, 4096), _log(rng, 16, 4096) | 1])
        most = 24_000_000 if kind == "conv_train" else 6_000_000
        L = _log(rng, 1, min(32768, most // D))
        B = _log(rng, 1, max(1, min(32, most // (D * L))))
        return _conv(None, kind, B, L, D, rng.choice([2, 3, 4, 4]), dtype, state=kind == "conv" and rng.random() < 0.5, ragged=rng.random() < 0.4 and L > 8)
    N = rng.choice([16, 16, 16, 8, 32, 64, 12])
    if kind == "step":
        D = rng.choice([384, 768, 1024, 1536, 2048])
        return _step(None, _log(rng, 1, max(1, 256 * 1536 * 16 // (D * max(N, 16)))), D, N, rng.choice([2, 3, 4, 4]), dtype)
    G = rng.choice([1, 1, 2, 4])
    D = G * rng.choice([96, 192, 256, 384, _log(rng, 8, 400)])
    most = (24_000_000 if kind == "scan" else 8_000_000) * 16 // max(N, 16)
    L = _log(rng, 17, min(16384, most // D))
    B = _log(rng, 1, max(1, min(16, most // (D * L))))
    return _scan(None, kind, B, L, D, N, G, dtype, gate=rng.random() < 0.7, state=kind == "scan" and rng.random() < 0.5, ragged=rng.random() < 0.4)


def _lens(case):
    """Live tokens of each row of a ragged batch: from half the length to all of it."""
    B, L = case["B"], case["L"]
    return [L - (L // 2) * i // B if case.get("ragged") else L for i in range(B)]


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind in ("norm_fp8", "norm_train"):
        rows, dim = case["rows"], case["dim"]
        x, r = _TYPES[case["x"]], _TYPES[case["r"]]
        # a layer's output, and a residual stream with channels of different scales
        s = {"x": randn(rows, dim).to(x), "residual": (randn(rows, dim) * (0.5 + 2 * randn(dim).abs())).to(r), "weight": 1 + 0.2 * randn(dim)}
        if kind == "norm_train":
            s["dy"], s["dr"] = randn(rows, dim).to(x), randn(rows, dim).to(r)
        return s
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        a, a_scale = _quantize(randn(M, K) * (0.5 + rand(M, 1)), 1)
        b, b_scale = _quantize(randn(N, K) * K ** -0.5, _BLOCK)
        return {"a": a, "a_scale": a_scale, "b": b, "b_scale": b_scale}
    B, L, D = case["B"], case["L"], case["D"]
    t = _TYPES[case["dtype"]]
    s = {"mask": None}
    if case.get("ragged"):
        lens = torch.tensor(_lens(case), device="cuda")[torch.randperm(B, generator=g, device="cuda")]
        s["mask"] = torch.arange(L, device="cuda")[None, :] < lens[:, None]
    if kind in ("conv", "conv_train", "step"):
        W = case["W"]
        # x is one half of a projection's [B, L, 2 D] output
        s["x"] = randn(B, L, 2 * D).to(t)[..., :D]
        s["weight"], s["bias"] = randn(D, W) * W ** -0.5, 0.1 * randn(D)
        s["window"] = randn(B, W - 1, D).to(t) if kind == "step" or case["state"] else None
        if kind == "conv_train":
            s["dout"] = randn(B, L, D).to(t)
        if kind != "step":
            return s
    N, G = case["N"], case["G"]
    s["u"] = torch.nn.functional.silu(randn(B, L, D)).to(t)
    # step sizes from 0.001 to 0.1, each channel with a mean of its own
    size = torch.exp(rand(D) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s["dt_bias"] = size + torch.log(-torch.expm1(-size))
    s["dt"] = (0.5 * randn(B, L, D)).to(t)
    s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * torch.exp(0.1 * randn(D, N))
    both = randn(B, L, G, 2 * N).to(t)  # one projection's output
    s["Bm"], s["C"] = both[..., :N], both[..., N:]
    s["D"] = 1 + 0.1 * randn(D)
    s["z"] = randn(B, L, 2 * D).to(t)[..., D:] if case.get("gate", True) else None
    s["state"] = 0.5 * randn(B, D, N) if kind == "step" or case["state"] else None
    if kind == "scan_train":
        s["dout"] = randn(B, L, D).to(t)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["kind"] = case["kind"]
    if case["kind"] == "matmul":
        s["out_dtype"] = _TYPES[case["dtype"]]
    if case["kind"] == "step":
        # a serving loop's buffers, refilled between steps, and its handles on them
        s["conv_out"], s["out"] = torch.empty_like(s["u"]), torch.empty_like(s["u"])
        if own:
            ops = _ops()
            s["conv_step"] = ops.CausalConvStep(s["x"], s["weight"], s["bias"], s["conv_out"], s["window"], activation="silu")
            s["scan_step"] = ops.SelectiveScanStep(s["u"], s["dt"], s["A"], s["Bm"], s["C"], s["out"], s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
    return s


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _quantize(x, rows):
    """e4m3 values and their scales, one for each `rows` x 128 of [M, K]: scale = amax / 448, value = x / scale."""
    M, K = x.shape
    m, k = -(-M // rows), -(-K // _BLOCK)
    full = torch.zeros(m * rows, k * _BLOCK, device=x.device)
    full[:M, :K] = x
    full = full.reshape(m, rows, k, _BLOCK)
    scale = full.abs().amax((1, 3)).clamp_min(1e-30) / _TOP
    q = (full / scale[:, None, :, None]).clamp(-_TOP, _TOP).reshape(m * rows, k * _BLOCK)[:M, :K]
    return q.contiguous().to(torch.float8_e4m3fn), scale


def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))


def _plain_conv(x, w, b, window, mask):
    """Float32; a masked token counts as 0 and gives 0. Returns the outputs and the window behind the last live token."""
    L, W = x.shape[1], w.shape[1]
    if mask is not None:
        x = torch.where(mask[..., None], x, torch.zeros_like(x))
    first = torch.zeros_like(x[:, :1]).expand(-1, W - 1, -1) if window is None else window
    full = torch.cat([first, x], 1)
    y = b + sum(w[:, j] * full[:, j:j + L] for j in range(W))
    y = _silu(y)
    if mask is None:
        return y, full[:, L:]
    y = torch.where(mask[..., None], y, torch.zeros_like(y))
    last = (mask * torch.arange(1, L + 1, device=x.device)).amax(1)
    at = last[:, None] + torch.arange(W - 1, device=x.device)
    return y, full.gather(1, at[..., None].expand(-1, -1, x.shape[2]))


def _plain_scan(u, dt, A, Bm, C, D, z, dt_bias, mask, h):
    """Float32: pieces of the sequence side by side, token by token, then joined; exact zeros where a token is masked."""
    B, L, Dn = u.shape
    N, G = A.shape[1], Bm.shape[2]
    dt = _softplus(dt + dt_bias)
    if mask is not None:
        live = mask[..., None]
        u, dt = (torch.where(live, x, torch.zeros_like(x)) for x in (u, dt))
        Bm, C = (torch.where(live[..., None], x, torch.zeros_like(x)) for x in (Bm, C))
    T = 1 << ((L - 1).bit_length() + 1) // 2  # about the root of L
    n = -(-L // T)
    pad = n * T - L
    uc, dtc = (torch.nn.functional.pad(x, (0, 0, 0, pad)).reshape(B, n, T, G, Dn // G, 1) for x in (u, dt))
    Bc, Cc = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)).reshape(B, n, T, G, 1, N) for x in (Bm, C))
    Ag = A.reshape(G, Dn // G, N)
    local, own_y = torch.zeros(B, n, G, Dn // G, N, device=u.device), []
    for t in range(T):
        local = torch.exp(dtc[:, :, t] * Ag) * local + dtc[:, :, t] * uc[:, :, t] * Bc[:, :, t]
        own_y.append((local * Cc[:, :, t]).sum(-1))
    since = dtc.cumsum(2)
    whole = torch.exp(since[:, :, -1] * Ag)
    carried = torch.zeros(B, G, Dn // G, N, device=u.device) if h is None else h.reshape(B, G, Dn // G, N)
    starts = []
    for c in range(n):
        starts.append(carried)
        carried = whole[:, c] * carried + local[:, c]
    starts = torch.stack(starts, 1)
    y = torch.stack([own_y[t] + (torch.exp(since[:, :, t] * Ag) * starts * Cc[:, :, t]).sum(-1) for t in range(T)], 2)
    y = y.reshape(B, n * T, Dn)[:, :L] + D * u
    if z is not None:
        y = y * _silu(z)
    if mask is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    return y, carried.reshape(B, Dn, N)


def _plain_step(s):
    t = s["x"].dtype
    W = s["weight"].shape[1]
    full = torch.cat([s["window"], s["x"]], 1)
    y = _silu((full.float() * s["weight"].t()).sum(1, keepdim=True) + s["bias"])
    s["conv_out"].copy_(y.to(t))
    s["window"].copy_(full[:, full.shape[1] - W + 1:])
    dt = _softplus(s["dt"].float() + s["dt_bias"])[:, 0, :, None]
    u, z = s["u"].float(), s["z"].float()
    h = torch.exp(dt * s["A"]) * s["state"] + dt * u[:, 0, :, None] * s["Bm"].float()[:, 0]
    s["state"].copy_(h)
    y = (h * s["C"].float()[:, 0]).sum(-1)[:, None] + s["D"] * u
    s["out"].copy_((y * _silu(z)).to(t))
    return s["conv_out"], s["window"], s["out"], s["state"]


def _plain_norm(s):
    t = s["x"].dtype
    r = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
    rf = r.float()
    rms = (rf.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xh = rf * rms
    if s["kind"] == "norm_fp8":
        return _quantize(xh * s["weight"], 1) + (r,)
    dy = s["dy"].float()
    gw = dy * s["weight"]
    dr = rms * (gw - xh * (gw * xh).mean(-1, keepdim=True)) + s["dr"].float()
    return (xh * s["weight"]).to(t), r, dr.to(t), dr.to(r.dtype), (dy * xh).sum(0)


def _plain_matmul(s):
    (M, K), N = s["a"].shape, s["b"].shape[0]
    a = s["a"].float() * s["a_scale"].repeat_interleave(_BLOCK, 1)[:, :K]
    b = s["b"].float() * s["b_scale"].repeat_interleave(_BLOCK, 0)[:N].repeat_interleave(_BLOCK, 1)[:, :K]
    return (a @ b.t()).to(s["out_dtype"])


_SCAN = ("u", "dt", "A", "Bm", "C", "D", "z", "dt_bias")


def _run_plain(s):
    kind = s["kind"]
    if kind in ("norm_fp8", "norm_train"):
        return _plain_norm(s)
    if kind == "matmul":
        return _plain_matmul(s)
    if kind == "step":
        return _plain_step(s)
    if kind in ("conv", "conv_train"):
        t = s["x"].dtype
        window = None if s["window"] is None else s["window"].float()
        if kind == "conv":
            y, window = _plain_conv(s["x"].float(), s["weight"], s["bias"], window, s["mask"])
            return y.to(t), window.to(t)
        leaves = [s[n].detach().float().requires_grad_(True) for n in ("x", "weight", "bias")]
        y, _ = _plain_conv(*leaves, window, s["mask"])
        dx, dw, db = torch.autograd.grad(y, leaves, s["dout"].float())
        return y.detach().to(t), dx.to(t), dw, db
    t = s["u"].dtype
    if kind == "scan":
        y, h = _plain_scan(*(None if s[n] is None else s[n].float() for n in _SCAN), s["mask"], s["state"])
        return (y.to(t), h) if s["state"] is not None else y.to(t)
    leaves = {n: s[n].detach().float().requires_grad_(True) for n in _SCAN if s[n] is not None}
    y, _ = _plain_scan(*(leaves.get(n) for n in _SCAN), s["mask"], None)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["dout"].float())))
    return (y.detach().to(t),) + tuple(grads[n].to(s[n].dtype) for n in _SCAN if n in grads)


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    ops = _ops()
    kind = s["kind"]
    if kind == "norm_fp8":
        return ops.rms_norm_fp8(s["x"], s["weight"], 1e-5, residual=s["residual"])
    if kind == "norm_train":
        y, r = ops.rms_norm(s["x"], s["weight"], 1e-5, residual=s["residual"])
        dx, dres, dw = ops.rms_norm_backward(s["dy"], r, s["weight"], 1e-5, dresidual=s["dr"])
        return y, r, dx, dres, dw
    if kind == "matmul":
        return ops.scaled_matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], out_dtype=s["out_dtype"])
    if kind == "step":
        s["conv_step"].step()
        s["scan_step"].step()
        return s["conv_out"], s["window"], s["out"], s["state"]
    if kind in ("conv", "conv_train"):
        y, window = ops.causal_conv_forward(s["x"], s["weight"], s["bias"], activation="silu", mask=s["mask"], state=s["window"], return_state=kind == "conv")
        if kind == "conv":
            return y, window
        dx, dw, db, _ = ops.causal_conv_backward(s["x"], s["weight"], s["dout"], s["bias"], activation="silu", mask=s["mask"])
        return y, dx, dw, db
    more = {"D": s["D"], "z": s["z"], "dt_bias": s["dt_bias"], "mask": s["mask"]}
    if kind == "scan":
        y, h = ops.selective_scan_forward(s["u"], s["dt"], s["A"], s["Bm"], s["C"], **more, state=s["state"], return_state=s["state"] is not None)
        return (y, h) if s["state"] is not None else y
    handover = ops.ScanHandover()
    y, _ = ops.selective_scan_forward(s["u"], s["dt"], s["A"], s["Bm"], s["C"], **more, handover=handover)
    g = ops.selective_scan_backward(s["u"], s["dt"], s["A"], s["Bm"], s["C"], s["dout"], **more, handover=handover)
    grads = {"u": g.du, "dt": g.ddt, "A": g.dA, "Bm": g.dB, "C": g.dC, "D": g.dD, "z": g.dz, "dt_bias": g.ddt_bias}
    return (y,) + tuple(grads[n] for n in _SCAN if s[n] is not None)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------- the work
def work(case):
    kind = case["kind"]
    if kind in ("norm_fp8", "norm_train"):
        n, x, r = case["rows"] * case["dim"], _SIZE[case["x"]], _SIZE[case["r"]]
        if kind == "norm_fp8":
            return {"bytes": n * (x + r + r + 1) + 4 * case["rows"] * -(-case["dim"] // _BLOCK) + 4 * case["dim"], "flops": 7 * n}
        # forward: x, residual in, r, y out; backward: dy, r, dr in, dx, dresidual out
        return {"bytes": n * (x + r + r + x + x + r + r + x + r) + 12 * case["dim"], "flops": 17 * n}
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        k = -(-K // _BLOCK)
        return {"bytes": M * K + N * K + 4 * k * (M + -(-N // _BLOCK)) + M * N * _SIZE[case["dtype"]], "flops": 2 * M * N * K}
    B, L, D, t = case["B"], case["L"], case["D"], _SIZE[case["dtype"]]
    live = sum(_lens(case))
    mask = B * L if case.get("ragged") else 0
    conv = scan = {"bytes": 0, "flops": 0}
    if "W" in case:
        W = case["W"]
        into, out, window = live * D * t, B * L * D * t, (2 if case.get("state", True) else 0) * B * (W - 1) * D * t
        flops = live * D * (2 * W + 4)
        if kind == "conv_train":
            conv = {"bytes": 3 * into + 2 * out + D * (W + 1) * 12 + mask, "flops": 4 * flops}
        else:
            conv = {"bytes": into + out + window + D * (W + 1) * 4 + mask, "flops": flops}
    if "N" in case:
        N, G = case["N"], case["G"]
        gate = case.get("gate", True)
        into = live * (D * (3 if gate else 2) + 2 * G * N) * t  # u, dt, z, B, C of the live tokens
        out, states, weights = B * L * D * t, (2 if case.get("state", True) else 0) * B * D * N * 4, (D * N + 2 * D) * 4
        flops = live * D * (7 * N + 12)  # an exponential and six operations a state
        if kind == "scan_train":
            grads = B * L * (D * (3 if gate else 2) + 2 * G * N) * t
            scan = {"bytes": 2 * into + out + live * D * t + grads + 3 * weights + mask, "flops": 4 * flops}
        else:
            scan = {"bytes": into + out + states + weights + mask, "flops": flops}
    return {n: conv[n] + scan[n] for n in ("bytes", "flops")}


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _sigmoid64(x):
    return torch.where(x >= 0, 1 / (1 + torch.exp(-x.abs())), 1 - 1 / (1 + torch.exp(-x.abs())))


def _exact_conv(s, dout):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    (B, L, D), W = x.shape, w.shape[1]
    live = torch.ones(B, L, device=x.device, dtype=torch.float64) if s["mask"] is None else s["mask"].double()
    past = torch.zeros(B, W - 1, D, device=x.device, dtype=torch.float64)
    if s["window"] is not None:
        past = s["window"].double()
    seen = torch.empty(B, W - 1 + L, D, device=x.device, dtype=torch.float64)
    seen[:, :W - 1], seen[:, W - 1:] = past, x * live[..., None]
    pre = b.expand(B, L, D).clone()
    for j in range(W):
        pre += seen.narrow(1, j, L) * w[:, j]
    sig = _sigmoid64(pre)
    y = pre * sig * live[..., None]
    if dout is None:
        ends = [int(v.nonzero().max()) + 1 if bool(v.any()) else 0 for v in live]
        return y, torch.stack([seen[i, e:e + W - 1] for i, e in enumerate(ends)])
    dpre = dout.double() * live[..., None] * sig * (1 + pre * (1 - sig))
    dseen, dw = torch.zeros_like(seen), torch.empty_like(w)
    for j in range(W):
        dseen.narrow(1, j, L).add_(dpre * w[:, j])
        dw[:, j] = (dpre * seen.narrow(1, j, L)).sum((0, 1))
    return y, dseen[:, W - 1:] * live[..., None], dw, dpre.sum((0, 1))


def _exact_scan(s, dout):
    """Token by token; the gradients from the adjoint recurrence."""
    B, L, D = s["u"].shape
    A = s["A"].double()
    group = torch.arange(D, device=A.device) // (D // s["Bm"].shape[2])
    m = torch.ones(B, L, 1, device=A.device, dtype=torch.float64) if s["mask"] is None else s["mask"].double()[..., None]
    u, z = s["u"].double(), None if s["z"] is None else s["z"].double()
    raw = s["dt"].double() + s["dt_bias"].double()
    dt = (raw.clamp_min(0) + torch.log1p(torch.exp(-raw.abs()))) * m
    Bm, C = s["Bm"].double(), s["C"].double()
    h = torch.zeros(B, D, A.shape[1], device=A.device, dtype=torch.float64) if s["state"] is None else s["state"].double()
    y = torch.empty(B, L, D, device=A.device, dtype=torch.float64)
    kept = []
    for t in range(L):
        if dout is not None:
            kept.append(h)
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * Bm[:, t, group]
        y[:, t] = torch.einsum("bdn,bdn->bd", h, C[:, t, group])
    y = (y + s["D"].double() * u) * m
    gate = 1.0 if z is None else z * _sigmoid64(z)
    if dout is None:
        return y * gate, h
    do = dout.double() * m
    dy = do * gate
    du, ddt = s["D"].double() * dy, torch.zeros_like(dt)
    dA, dB, dC = torch.zeros_like(A), torch.zeros_like(Bm), torch.zeros_like(C)
    adj, ones = torch.zeros_like(h), torch.ones(B, D, A.shape[1], device=A.device, dtype=torch.float64)
    for t in reversed(range(L)):
        Bt, d = Bm[:, t, group], dt[:, t, :, None]
        before = torch.exp(d * A) * kept.pop()
        now = before + d * u[:, t, :, None] * Bt
        adj = adj + dy[:, t, :, None] * C[:, t, group]
        dC[:, t].index_add_(1, group, now * dy[:, t, :, None])
        dB[:, t].index_add_(1, group, adj * d * u[:, t, :, None])
        into = (adj * Bt).sum(-1)
        du[:, t] += dt[:, t] * into
        ddt[:, t] = u[:, t] * into + (adj * before * A).sum(-1)
        dA += (adj * before * d).sum(0)
        adj = adj * torch.exp(d * A) * ones
    draw_dt = ddt * _sigmoid64(raw) * m
    got = {"u": du, "dt": draw_dt, "A": dA, "Bm": dB, "C": dC, "D": (dy * u).sum((0, 1)), "dt_bias": draw_dt.sum((0, 1))}
    if z is not None:
        sig = _sigmoid64(z)
        got["z"] = do * y * sig * (1 + z * (1 - sig))
    live = m[..., None]
    got["u"], got["Bm"], got["C"] = got["u"] * m, got["Bm"] * live, got["C"] * live
    return (y * gate,) + tuple(got[n] for n in _SCAN if n in got)


def _exact_quantized(y):
    rows, dim = y.shape
    parts = [y[:, at:at + _BLOCK] for at in range(0, dim, _BLOCK)]
    scale = torch.stack([p.abs().max(1).values.clamp_min(1e-30) / _TOP for p in parts], 1)
    q = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], 1)
    # to the nearest of 4 significant bits, with a step of 2^-9 below 2^-6; ties to even
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(q / step) * step, scale


def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind in ("norm_fp8", "norm_train"):
        r = (s["x"].double() + s["residual"].double()).to(s["residual"].dtype)
        r64 = r.double()
        root = torch.sqrt(r64.pow(2).sum(-1) / case["dim"] + 1e-5)[:, None]
        y = r64 / root * s["weight"].double()
        if kind == "norm_fp8":
            return _exact_quantized(y) + (r64,)
        dy, w = s["dy"].double(), s["weight"].double()
        n = r64 / root
        dr = (dy * w - n * ((dy * w * n).sum(-1) / case["dim"])[:, None]) / root + s["dr"].double()
        return y, r64, dr, dr, (dy * n).sum(0)
    if kind == "matmul":
        if case["M"] * case["N"] * case["K"] > 100_000_000_000:
            return None
        (M, K), N = s["a"].shape, s["b"].shape[0]
        out = torch.zeros(M, N, device="cuda", dtype=torch.float64)
        for i, at in enumerate(range(0, K, _BLOCK)):
            rows = s["b_scale"][:, i].double()[torch.arange(N, device="cuda") // _BLOCK]
            part = s["a"][:, at:at + _BLOCK].double() @ s["b"][:, at:at + _BLOCK].double().t()
            out += part * s["a_scale"][:, i].double()[:, None] * rows
        return out
    if kind in ("conv", "conv_train"):
        return _exact_conv(s, s.get("dout"))
    if kind == "step":
        W = case["W"]
        seen = torch.cat([s["window"], s["x"]], 1).double()
        pre = torch.einsum("bwd,dw->bd", seen, s["weight"].double()) + s["bias"].double()
        got = _exact_scan(s, None)
        return (pre * _sigmoid64(pre))[:, None], seen[:, 1:W], got[0], got[1]
    got = _exact_scan(s, s.get("dout"))
    return got if kind == "scan_train" or case["state"] else got[0]
