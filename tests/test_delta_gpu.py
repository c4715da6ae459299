"""The gated delta rule (ops.gated_delta_forward / _backward, GatedDeltaStep)
against its definition in float64 (delta_reference.py).

Tolerances, relative in the 2-norm over a tensor. An output rounded once is off
by at most half a step, u = eps / 2 of its type. Inside, 16-bit inputs' operands
are rounded to two bf16 planes: at most 2^-16 and about 2.7e-6 in the mean
square; about six such roundings lie between the inputs and any result, each
fresh to every element: 7e-6, and a factor of 4 for how the recurrence passes
errors on: 3e-5. float32 inputs go through three planes (2^-24) and float32
sums of up to 64 products (64 x 2^-24 at most, 8 x 2^-24 in the mean square):
2e-6 with the same factor; the token-recurrent kernel is float32 throughout.
Inputs as the rule meets them: unit keys, beta in (0, 1), decay below 1.
"""
import math

import pytest
import torch

import delta_reference as ref
from subq_audio import _capi, ops

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def tol(out_dtype, in_dtype):
    inside = 2e-6 if in_dtype == torch.float32 else 3e-5
    return inside + (torch.finfo(out_dtype).eps / 2 if out_dtype != torch.float32 else 0.0)


def rel(a, b):
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    n = float(b.norm())
    d = float((a - b).norm())
    return d / n if n > 0 else d


def inputs(B, H, Hq, Hk, Hv, N, d, e, dtype, seed=0, layout="bnhd", mask=None, state=True, decay=True):
    g = torch.Generator().manual_seed(seed)

    def heads(h, w, unit=False):
        x = torch.randn(B, N, h, w, generator=g) if layout != "bhnd" else torch.randn(B, h, N, w, generator=g)
        if unit:
            x = x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)
        x = x.to(T[dtype])
        if layout == "odd":  # rows that start on no 16-byte boundary
            wide = torch.zeros(B, N, h, w + 3, dtype=T[dtype])
            wide[..., 1:w + 1] = x
            return wide.cuda()[..., 1:w + 1].transpose(1, 2)
        return x.cuda().transpose(1, 2) if layout == "bnhd" else x.cuda()

    q, k, v, do = heads(Hq, d, True), heads(Hk, d, True), heads(Hv, e), heads(H, e)
    beta = torch.sigmoid(torch.randn(B, N, H, generator=g)).cuda().transpose(1, 2)
    lg = torch.zeros(B, H, N).cuda()
    if decay:
        lg = -torch.nn.functional.softplus(-(torch.randn(B, N, H, generator=g) + 2)).cuda().transpose(1, 2)
    S0 = 0.5 * torch.randn(B, H, d, e, generator=g).cuda() if state else None
    dS = torch.randn(B, H, d, e, generator=g).cuda()
    m = None
    if mask == "tail":
        lens = torch.tensor([max(0, N - 1 - 37 * i) for i in range(B)])
        m = (torch.arange(N)[None] < lens[:, None]).cuda()
    elif mask == "random":
        m = (torch.rand(B, N, generator=g) < 0.6).cuda()
    elif mask == "holes":  # whole chunks without a live token, and a row without any
        m = torch.ones(B, N, dtype=torch.bool)
        m[:, 64:128] = False
        m[-1] = False
        m = m.cuda()
    return q, k, v, do, beta, lg, S0, dS, m


def poison(x, m):
    """NaN, infinities and the type's lowest value at the masked tokens."""
    if m is None:
        return x
    x = x.clone()
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(x.dtype).min], dtype=x.dtype, device=x.device)
    fill = bad[torch.arange(x.numel(), device=x.device) % 4].reshape(x.shape)
    mm = ~m.bool()[:, None, :]
    return torch.where(mm if x.dim() == 3 else mm[..., None], fill, x)


CASES = [
    # B, H, Hq, Hk, Hv, N, d, e, dtype, layout, mask, state
    (1, 1, 1, 1, 1, 1, 64, 64, "bf16", "bnhd", None, True),
    (2, 3, 3, 3, 3, 17, 64, 64, "bf16", "bnhd", None, False),
    (2, 2, 2, 2, 2, 64, 64, 64, "bf16", "bhnd", None, True),
    (2, 2, 2, 2, 2, 65, 64, 64, "fp16", "bnhd", None, True),
    (3, 4, 4, 2, 2, 200, 64, 64, "bf16", "bnhd", "tail", True),
    (2, 4, 2, 2, 4, 130, 64, 64, "fp16", "bnhd", "random", False),
    (2, 4, 4, 1, 2, 191, 64, 64, "fp32", "bnhd", "holes", True),
    (1, 2, 2, 2, 2, 333, 128, 128, "bf16", "bnhd", None, True),
    (2, 2, 1, 2, 1, 100, 128, 64, "fp32", "bhnd", "random", True),
    (1, 2, 2, 2, 2, 150, 128, 128, "fp16", "bnhd", "tail", True),
    (2, 2, 2, 2, 2, 129, 80, 48, "bf16", "odd", "random", True),
    (2, 2, 2, 2, 2, 70, 33, 17, "fp32", "odd", None, True),
    (1, 1, 1, 1, 1, 90, 5, 1, "fp32", "bhnd", "tail", True),
    (1, 2, 2, 2, 2, 66, 64, 256, "bf16", "bnhd", None, True),
    (1, 2, 2, 2, 2, 1000, 64, 64, "bf16", "bnhd", None, False),
]
IDS = ["-".join(str(x) for x in c) for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("path", ["exact", "chunked"])
def test_forward(case, path):
    B, H, Hq, Hk, Hv, N, d, e, dtype, layout, mask, state = case
    q, k, v, _, beta, lg, S0, _, m = inputs(B, H, Hq, Hk, Hv, N, d, e, dtype, seed=N + d, layout=layout, mask=mask, state=state)
    scale = d ** -0.5
    o_ref, S_ref = ref.forward(q, k, v, beta, lg, m, scale, S0)
    o, S = ops.gated_delta_forward(poison(q, m), poison(k, m), poison(v, m), poison(beta, m), log_gamma=poison(lg, m), mask=m,
                                   state=S0, return_state=True, path=path)
    assert ops.last_path() == path
    assert o.dtype == q.dtype and S.dtype == torch.float32
    assert rel(o, o_ref) < tol(o.dtype, q.dtype)
    assert rel(S, S_ref) < tol(S.dtype, q.dtype)
    if m is not None:
        assert bool((o.transpose(1, 2)[~m] == 0).all())


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("carried", [True, False])
def test_backward(case, carried):
    B, H, Hq, Hk, Hv, N, d, e, dtype, layout, mask, state = case
    q, k, v, do, beta, lg, S0, dS, m = inputs(B, H, Hq, Hk, Hv, N, d, e, dtype, seed=N + d, layout=layout, mask=mask, state=state)
    scale = d ** -0.5
    want = ref.gradients(q, k, v, beta, lg, m, scale, S0, do, dS if state else None)
    q, k, v, do, beta, lg = (poison(x, m) for x in (q, k, v, do, beta, lg))
    ho = ops.DeltaHandover() if carried else None
    if carried:
        ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, handover=ho)
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS if state else None,
                                   need_dlog_gamma=True, need_dstate=True, handover=ho)
    for name, a, b in zip(("dq", "dk", "dv", "dbeta", "dlog_gamma", "dstate"), got, want):
        assert rel(a, b) < tol(a.dtype, q.dtype), name
        if m is not None and name != "dstate":
            assert bool((a.transpose(1, 2)[~m] == 0).all()), name


LONG = [(1, 2, 2, 1, 2, 3000, 64, 64, "bf16", None), (1, 1, 1, 1, 1, 5001, 64, 96, "fp16", "tail"),
        (2, 1, 1, 1, 1, 4097, 100, 40, "fp32", "random"), (1, 3, 3, 3, 3, 2950, 128, 128, "bf16", "random")]


@pytest.mark.parametrize("case", LONG, ids=["-".join(str(x) for x in c) for c in LONG])
def test_long_and_few_sequences(case):
    """Sequences that are cut into segments walked side by side, then joined; the backward from their handover and
    from its own."""
    B, H, Hq, Hk, Hv, N, d, e, dtype, mask = case
    q, k, v, do, beta, lg, S0, dS, m = inputs(B, H, Hq, Hk, Hv, N, d, e, dtype, seed=N, mask=mask)
    if mask == "random":
        m[:, 640:1024] = False  # whole chunks, one of them the first of a segment
    scale = d ** -0.5
    with torch.no_grad():
        o_ref, S_ref = ref.forward(q, k, v, beta, lg, m, scale, S0)
    ho = ops.DeltaHandover()
    o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, return_state=True)
    assert ops.last_launches() == 4
    o2, S2 = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, return_state=True, handover=ho)
    assert torch.equal(o, o2) and torch.equal(S, S2)
    assert rel(o, o_ref) < tol(o.dtype, q.dtype) and rel(S, S_ref) < tol(S.dtype, q.dtype)
    want = ref.gradients(q, k, v, beta, lg, m, scale, S0, do, dS)
    runs = [ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True,
                                     need_dstate=True, handover=h) for h in (ho, None)]
    for name, a, b, w in zip(("dq", "dk", "dv", "dbeta", "dlog_gamma", "dstate"), *runs, want):
        assert torch.equal(a, b), name
        assert rel(a, w) < tol(a.dtype, q.dtype), name


def test_backward_is_reproducible_and_equal_with_and_without_the_handover():
    q, k, v, do, beta, lg, S0, dS, m = inputs(2, 4, 4, 2, 2, 300, 64, 64, "bf16", mask="tail")
    ho = ops.DeltaHandover()
    ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, handover=ho)
    runs = [ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True,
                                     need_dstate=True, handover=h) for h in (ho, ho, None)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_gradients_against_differences():
    """Central differences of the kernels' own float32 forward along random directions. The loss
    <o, do> + <S, dS> is smooth; a step h = 2^-6 leaves h^2 ~ 2.4e-4 of its third derivatives along a
    unit direction and rounding 2^-20 |loss| / h; 1 % covers both."""
    q, k, v, do, beta, lg, S0, dS, _ = inputs(1, 2, 2, 1, 2, 100, 32, 32, "fp32", seed=5)

    def loss(q, k, v, beta, lg, S0):
        o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, state=S0, return_state=True)
        return float((o.double() * do.double()).sum() + (S.double() * dS.double()).sum())

    leaves = [q, k, v, beta, lg, S0]
    grads = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True)
    for i, g in enumerate(grads):
        u = g / g.norm()  # the steepest direction: no cancellation
        h = 2.0 ** -6
        up, down = ([x + s * h * u if j == i else x for j, x in enumerate(leaves)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(slope - float(g.norm())) < 0.01 * float(g.norm()), i


def test_strong_and_absent_decay():
    """gamma = 0 (log gamma = -inf) restarts the state; no log_gamma and beta None are 1."""
    q, k, v, do, beta, lg, S0, dS, _ = inputs(1, 2, 2, 2, 2, 140, 64, 64, "fp32", seed=9)
    lg = lg.clone()
    lg[:, :, [0, 50, 51, 100]] = -math.inf
    lg[:, :, 70] = -500.0
    safe = lg.clamp_min(-800.0)  # exp is 0 in float64 too
    for path in ("exact", "chunked"):
        o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, state=S0, return_state=True, path=path)
        o_ref, S_ref = ref.forward(q, k, v, beta, safe, None, 64 ** -0.5, S0)
        assert rel(o, o_ref) < 2e-6 and rel(S, S_ref) < 2e-6
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True)
    want = ref.gradients(q, k, v, beta, safe, None, 64 ** -0.5, S0, do, dS)
    for a, b in zip(got, want):
        assert rel(a, b) < 2e-6
    ones, zeros = torch.ones_like(beta), torch.zeros_like(beta)
    for path in ("exact", "chunked"):
        o, S = ops.gated_delta_forward(q, k, v, None, state=S0, return_state=True, path=path)
        o_ref, S_ref = ref.forward(q, k, v, ones, zeros, None, 64 ** -0.5, S0)
        # with beta 1, random unit keys and no decay nothing is forgotten but what is overwritten: errors of
        # all 140 tokens stay (12 x in the mean square rather than the factor of 4)
        assert rel(o, o_ref) < 6e-6 and rel(S, S_ref) < 6e-6


def test_equal_keys_and_zero_beta():
    """All keys equal with beta 1 (each token replaces the last), and beta 0 (the state stands still)."""
    q, k, v, do, beta, lg, S0, dS, _ = inputs(1, 1, 1, 1, 1, 96, 64, 64, "fp32", seed=4, decay=False)
    k = k[:, :, :1].expand_as(k)
    for b in (torch.ones_like(beta), torch.zeros_like(beta)):
        o, S = ops.gated_delta_forward(q, k, v, b, log_gamma=lg, state=S0, return_state=True, path="chunked")
        o_ref, S_ref = ref.forward(q, k, v, b, lg, None, 64 ** -0.5, S0)
        assert rel(o, o_ref) < 2e-6 and rel(S, S_ref) < 2e-6
        got = ops.gated_delta_backward(q, k, v, b, do, log_gamma=lg, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True)
        want = ref.gradients(q, k, v, b, lg, None, 64 ** -0.5, S0, do, dS)
        for name, x, y in zip(("dq", "dk", "dv", "dbeta", "dlg", "dS"), got, want):
            assert rel(x, y) < 6e-6, (name, float(b[0, 0, 0]))


@pytest.mark.parametrize("N", [0, 1, 40])
def test_empty_and_wholly_masked_calls(N):
    q, k, v, do, beta, lg, S0, dS, _ = inputs(2, 2, 2, 2, 2, N, 64, 64, "bf16")
    m = torch.zeros(2, N, dtype=torch.bool, device="cuda")
    for path in ("exact", "chunked"):
        o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, return_state=True, path=path)
        assert torch.equal(S, S0) and bool((o == 0).all())
        _, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, return_state=True, path=path)
        assert bool((S == 0).all())
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True,
                                   need_dstate=True)
    assert torch.equal(got[5], dS) and all(bool((g == 0).all()) for g in got[:5])
    e = torch.empty(0, 2, 5, 64, device="cuda", dtype=torch.bfloat16)
    o, S = ops.gated_delta_forward(e, e, e, None, return_state=True)
    assert o.shape == (0, 2, 5, 64) and S.shape == (0, 2, 64, 64)


@pytest.mark.parametrize("path,d,e", [("exact", 200, 200), ("exact", 256, 30), ("chunked", 128, 256), ("exact", 64, 64)])
def test_pieces_with_a_carried_state_equal_one_call(path, d, e):
    q, k, v, _, beta, lg, S0, _, m = inputs(2, 2, 2, 2, 2, 150, d, e, "fp32", mask="random")
    o_all, S_all = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, return_state=True, path=path)
    o_ref, S_ref = ref.forward(q, k, v, beta, lg, m, d ** -0.5, S0)
    assert rel(o_all, o_ref) < 2e-6 and rel(S_all, S_ref) < 2e-6
    S, outs = S0, []
    for a, b in ((0, 1), (1, 40), (40, 104), (104, 150)):
        o, S = ops.gated_delta_forward(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], beta[:, :, a:b], log_gamma=lg[:, :, a:b],
                                       mask=m[:, a:b], state=S, return_state=True)
        outs.append(o)
    assert rel(torch.cat(outs, 2), o_ref) < 2e-6 and rel(S, S_ref) < 2e-6


@pytest.mark.parametrize("dtype,d,e,Hkv,Tn", [("bf16", 64, 64, 4, 1), ("fp16", 128, 96, 2, 1), ("fp32", 256, 256, 1, 3),
                                              ("bf16", 33, 7, 4, 2), ("bf16", 64, 64, 2, 40)])
def test_step_over_preallocated_buffers(dtype, d, e, Hkv, Tn):
    B, H, steps = 3, 4, 5
    q, k, v, _, beta, lg, S0, _, _ = inputs(B, H, H, Hkv, Hkv, steps * Tn, d, e, dtype)
    qb, kb, vb = (torch.empty(B, x.shape[1], Tn, x.shape[3], dtype=x.dtype, device="cuda") for x in (q, k, v))
    bb, lb = (torch.empty(B, H, Tn, device="cuda") for _ in range(2))
    mask = torch.ones(B, Tn, dtype=torch.bool, device="cuda")
    out, S = torch.empty(B, H, Tn, e, dtype=q.dtype, device="cuda"), S0.clone()
    step = ops.GatedDeltaStep(qb, kb, vb, bb, out, S, log_gamma=lb, mask=mask)

    def fill(i):
        for dst, src in ((qb, q), (kb, k), (vb, v), (bb, beta), (lb, lg)):
            dst.copy_(src[:, :, i * Tn:(i + 1) * Tn])

    o_ref, S_ref = ref.forward(q, k, v, beta, lg, None, d ** -0.5, S0)
    outs = []
    for i in range(steps):
        fill(i)
        step.step()
        outs.append(out.clone())
    assert rel(torch.cat(outs, 2), o_ref) < tol(q.dtype, q.dtype) and rel(S, S_ref) < tol(torch.float32, q.dtype)
    # the same steps captured once and replayed, on another stream
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.step()
    S.copy_(S0)
    again = []
    for i in range(steps):
        fill(i)
        graph.replay()
        again.append(out.clone())
    assert torch.equal(torch.cat(again, 2), torch.cat(outs, 2))


def test_captured_training_step_and_two_streams():
    """Forward and backward captured together and replayed on new inputs, while the same operators run
    eagerly on another stream: each call's workspace is its own."""
    q, k, v, do, beta, lg, _, _, m = inputs(2, 4, 4, 2, 2, 300, 64, 64, "bf16", mask="tail")

    def run(q, k, v, do, beta, lg):
        ho = ops.DeltaHandover()
        o, _ = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, handover=ho)
        return (o,) + ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, need_dlog_gamma=True, handover=ho)[:5]

    fixed = [x.clone() for x in (q, k, v, do, beta, lg)]
    run(*fixed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(*fixed)
    q2, k2, v2, do2, beta2, lg2, *_ = inputs(2, 4, 4, 2, 2, 300, 64, 64, "bf16", seed=77)
    new = (q2, k2, v2, do2, beta2, lg2)
    for dst, src in zip(fixed, new):
        dst.copy_(src)
    want_new, want_old = run(*new), run(q, k, v, do, beta, lg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            eager = run(q, k, v, do, beta, lg)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want_new))
    assert all(torch.equal(a, b) for a, b in zip(eager, want_old))


def test_gate_forms_and_the_rows_behind_a_slice():
    """Numbers, [H] and stride-0 gates equal the tensor they stand for; memory around an output view stays."""
    q, k, v, do, beta, lg, S0, _, _ = inputs(2, 4, 4, 4, 4, 80, 64, 64, "bf16")
    for path in ("exact", "chunked"):
        per_head = torch.tensor([-0.1, -0.2, -0.3, 0.0], device="cuda")
        a = ops.gated_delta_forward(q, k, v, 0.5, log_gamma=per_head, path=path)[0]
        full = per_head.view(1, 4, 1).expand(2, 4, 80).contiguous()
        b = ops.gated_delta_forward(q, k, v, torch.full((2, 4, 80), 0.5, device="cuda"), log_gamma=full, path=path)[0]
        c = ops.gated_delta_forward(q, k, v, torch.full((2, 4, 80), 0.5, device="cuda", dtype=torch.bfloat16),
                                    log_gamma=full[:, :, :1], path=path)[0]
        assert torch.equal(a, b) and torch.equal(a, c)
        wide = torch.full((2, 4, 100, 72), 7.0, device="cuda", dtype=torch.bfloat16)
        ops.gated_delta_forward(q, k, v, 0.5, log_gamma=per_head, path=path, out=wide[:, :, 10:90, 4:68])
        assert torch.equal(wide[:, :, 10:90, 4:68], a)
        assert bool((wide[:, :, :10] == 7).all() and (wide[:, :, 90:] == 7).all() and (wide[..., :4] == 7).all()
                    and (wide[..., 68:] == 7).all())


def test_refusals():
    q, k, v, do, beta, lg, S0, dS, m = inputs(2, 4, 4, 2, 2, 40, 64, 64, "bf16", mask="tail")
    f = ops.gated_delta_forward
    with pytest.raises(RuntimeError, match="CUDA"):
        f(q.cpu(), k.cpu(), v.cpu(), None)
    with pytest.raises(TypeError, match="share one dtype"):
        f(q, k.float(), v, beta)
    with pytest.raises(TypeError, match="unsupported dtype"):
        f(q.double(), k.double(), v.double(), beta)
    for bad in (lambda: f(q, k[:, :, :20], v, beta), lambda: f(q, k[..., :32], v, beta), lambda: f(q[:, :3], k, v, beta),
                lambda: f(q, k, v, beta[:, :, :20]), lambda: f(q, k, v, beta, log_gamma=lg[:, :3]),
                lambda: f(q, k, v, beta, mask=m[:, :20]), lambda: f(q, k, v, beta, state=S0[:, :2]),
                lambda: f(q, k, v, beta, out=torch.empty_like(k)), lambda: f(q[0], k, v, beta),
                lambda: f(q, k, v, beta, path="tensorcore"), lambda: f(q, k, v, beta, path="fast"),
                lambda: f(q, k, v, beta, scale=math.inf),
                lambda: ops.gated_delta_backward(q, k, v, beta, do[:, :, :20])):
        with pytest.raises(ValueError):
            bad()
    big = torch.randn(1, 1, 20, 160, device="cuda")
    with pytest.raises(_capi.SubqError, match="head_dim"):
        f(big, big, big, None, path="chunked")
    with pytest.raises(_capi.SubqError, match="head_dim"):
        ops.gated_delta_backward(big, big, big, None, big)
    ho = ops.DeltaHandover()
    f(q, k, v, beta, handover=ho)
    with pytest.raises(ValueError, match="handover"):
        ops.gated_delta_backward(q[:, :, :30], k[:, :, :30], v[:, :, :30], beta[:, :, :30], do[:, :, :30], handover=ho)
    out, S = torch.empty(2, 4, 40, 64, device="cuda", dtype=torch.bfloat16), S0.clone()
    with pytest.raises(ValueError, match="float32"):
        ops.GatedDeltaStep(q, k, v, beta.bfloat16(), out, S)
    with pytest.raises(ValueError, match="contiguous float32"):
        ops.GatedDeltaStep(q, k, v, beta, out, S.half())
    with pytest.raises(ValueError, match="mask"):
        ops.GatedDeltaStep(q, k, v, beta, out, S, mask=m.float())


@pytest.mark.parametrize("d,e", [(64, 64), (100, 40)])
def test_state_in_place_where_a_sequence_is_cut_into_segments(d, e):
    """One segment's walk starts from the state that another one's overwrites at its end."""
    q, k, v, _, beta, lg, S0, _, _ = inputs(1, 4, 4, 4, 4, 4096, d, e, "bf16", seed=7)
    o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, state=S0, return_state=True)
    assert ops.last_launches() == 4
    state, out = S0.clone(), torch.empty_like(o)
    step = ops.GatedDeltaStep(q, k, v, beta, out, state, log_gamma=lg)
    for _ in range(3):
        state.copy_(S0)
        step.step()
        assert torch.equal(out, o) and torch.equal(state, S)


def test_buffers_that_do_not_belong_to_the_call_are_refused():
    q, k, v, do, beta, lg, _, _, _ = inputs(1, 2, 2, 2, 2, 100, 64, 64, "bf16")
    with pytest.raises(ValueError, match="o must not be"):
        ops.gated_delta_forward(q, k, v, beta, out=v)
    ho = ops.DeltaHandover()
    ops.gated_delta_forward(q, k, v, beta, handover=ho)
    for buf in (ho.buf[:-1], ho.buf.view(torch.int32), torch.empty(256, dtype=torch.uint8, device="cuda")):
        with pytest.raises(ValueError):
            torch.ops.subq_audio.gated_delta_bwd(q, k, v, beta, do, lg, None, None, None, 0.125, buf, False, False)
    ho.buf = ho.buf[::2]
    with pytest.raises(ValueError):
        ops.gated_delta_backward(q, k, v, beta, do, handover=ho)


@pytest.mark.parametrize("path", ["exact", "chunked"])
def test_offsets_beyond_32_bits(path):
    """Tokens 2^26 elements apart, heads interleaved: the last token's offset passes 2^31 elements."""
    N, step = 40, 1 << 26
    q, k, v, do, beta, lg, S0, dS, _ = inputs(1, 2, 2, 2, 2, N, 64, 64, "bf16", seed=3)
    buf = torch.empty((N - 1) * step + 1024, dtype=torch.bfloat16, device="cuda")

    def far(x, at):
        y = buf.as_strided(x.shape, (0, 64, step, 1), at)
        return y.copy_(x)

    fq, fk, fv, out, fdo = far(q, 0), far(k, 128), far(v, 256), far(v, 384), far(do, 512)
    args = dict(log_gamma=lg, state=S0)
    want, S = ops.gated_delta_forward(q, k, v, beta, return_state=True, path=path, **args)
    got, S2 = ops.gated_delta_forward(fq, fk, fv, beta, return_state=True, path=path, out=out, **args)
    assert torch.equal(want, got) and torch.equal(S, S2)
    if path == "chunked":
        runs = [ops.gated_delta_backward(*x, beta, g, dstate=dS, need_dlog_gamma=True, need_dstate=True, **args)
                for x, g in (((q, k, v), do), ((fq, fk, fv), fdo))]
        assert all(torch.equal(a, b) for a, b in zip(*runs))
        x, dy = fq[0, 0], fv[0, 0]  # [N, 64] rows, 2^26 apart
        assert torch.equal(ops.layer_norm(x), ops.layer_norm(x.contiguous()))
        assert all(torch.equal(a, b) for a, b in zip(ops.layer_norm_backward(dy, x), ops.layer_norm_backward(dy.contiguous(), x.contiguous())))


@pytest.mark.parametrize("d,e,N", [(1, 1, 70), (1, 33, 17), (33, 1, 130), (8, 256, 65)])
def test_smallest_heads(d, e, N):
    q, k, v, do, beta, lg, S0, dS, m = inputs(2, 3, 3, 1, 3, N, d, e, "bf16", seed=d + e, mask="random")
    want, S = ref.forward(q, k, v, beta, lg, m, d ** -0.5, S0)
    for path in ("exact", "chunked"):
        o, St = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, return_state=True, path=path)
        assert rel(o, want) < tol(o.dtype, q.dtype) and rel(St, S) < tol(St.dtype, q.dtype)
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True)
    for name, a, w in zip(("dq", "dk", "dv", "dbeta", "dlog_gamma", "dstate"), got, ref.gradients(q, k, v, beta, lg, m, d ** -0.5, S0, do, dS)):
        assert rel(a, w) < tol(a.dtype, q.dtype), name


def test_two_host_threads_at_once():
    import threading
    cases = [inputs(2, 4, 4, 2, 4, 700, 64, 64, "bf16", seed=s) for s in range(2)]

    def work(i, out):
        q, k, v, do, beta, lg, S0, dS, _ = cases[i]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                ho = ops.DeltaHandover()
                o, S = ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, state=S0, return_state=True, handover=ho)
                g = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, state=S0, dstate=dS, need_dlog_gamma=True,
                                             need_dstate=True, handover=ho)
                out[i] = (o, S) + g
        stream.synchronize()

    torch.cuda.synchronize()
    alone, both = [None, None], [None, None]
    for i in range(2):
        work(i, alone)
    threads = [threading.Thread(target=work, args=(i, both)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, both):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("N,d,e,dtype,dead", [(4096, 64, 64, "bf16", None), (2049, 128, 96, "bf16", (512, 1100)), (3333, 48, 80, "fp16", (0, 700)),
                                              (2500, 64, 64, "fp32", (1800, 2500)), (2500, 128, 128, "fp32", None)])
def test_gradients_where_the_walk_back_is_cut_into_segments(N, d, e, dtype, dead):
    q, k, v, do, beta, lg, S0, dS, _ = inputs(1, 2, 2, 1, 2, N, d, e, dtype, seed=N + d)
    m = torch.ones(1, N, dtype=torch.bool, device="cuda")
    if dead:
        m[:, dead[0]:dead[1]] = False
    ho = ops.DeltaHandover()
    ops.gated_delta_forward(q, k, v, beta, log_gamma=lg, mask=m, state=S0, handover=ho)
    got = ops.gated_delta_backward(q, k, v, beta, do, log_gamma=lg, mask=m, state=S0, dstate=dS, need_dlog_gamma=True, need_dstate=True,
                                   handover=ho)
    assert ops.last_launches() == 4 + 1  # states, join, walk, gradients; dk summed over its group
    want = ref.gradients(q, k, v, beta, lg, m, d ** -0.5, S0, do, dS)
    for name, a, w in zip(("dq", "dk", "dv", "dbeta", "dlog_gamma", "dstate"), got, want):
        assert rel(a, w) < tol(a.dtype, q.dtype), name
    none = ops.gated_delta_backward(q, k, v, beta, torch.zeros_like(do), log_gamma=lg, mask=m, state=S0, need_dlog_gamma=True, need_dstate=True)
    assert all(not x.any() for x in none)
