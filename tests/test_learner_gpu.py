"""The learner layers on the GPU, through the C ABI, against their definitions in 64 bits
(tests/learner_reference.py, where the bounds are derived), at the sizes, strides and masks where they can go wrong."""
from __future__ import annotations

import itertools

import pytest

import turbinator_c_b200 as tb
from tests import learner_reference as ref

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, tb.TB_TYPE_F32), "bf16": (torch.bfloat16, tb.TB_TYPE_BF16),
         "f16": (torch.float16, tb.TB_TYPE_F16)}
ACTS = {"none": tb.TB_ACT_NONE, "relu": tb.TB_ACT_RELU, "silu": tb.TB_ACT_SILU, "gelu": tb.TB_ACT_GELU}
NAN = float("nan")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(gen, *shape, scale=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda") * scale + mean


def _lay(v, kind, pad=0, shift=0):
    """`v` [a, b, c] as a slice of rows `pad` elements longer, `shift` elements into its buffer; NaN around it.
    Returns the view, the whole buffer."""
    a, b, c = v.shape
    buf = torch.full((a * b * (c + pad) + shift + 8,), NAN, dtype=kind, device="cuda")
    view = buf[shift:shift + a * b * (c + pad)].view(a, b, c + pad)[..., :c]
    view.copy_(v)
    return view, buf


def _untouched(view, buf, shift):
    """Everything of the buffer outside the view is still NaN."""
    a, b, c = view.shape
    wide = view.stride(1)
    inner = torch.zeros(buf.shape, dtype=torch.bool, device="cuda")
    inner[shift:shift + a * b * wide].view(a, b, wide)[..., :c] = True
    return bool(torch.isnan(buf[~inner]).all())


def _scratch(need):
    return torch.full((max(need, 1) + 16,), 0xA5, dtype=torch.uint8, device="cuda")


# ---- group norm ----

NORM_SHAPES = [
    # samples, positions, channels, groups, pad, shift
    (1, 1, 4, 1, 0, 0), (2, 1, 64, 2, 0, 0), (3, 7, 24, 8, 0, 0), (2, 256, 32, 8, 0, 0), (5, 100, 64, 64, 0, 0),
    (2, 33, 15, 5, 0, 0), (2, 33, 21, 3, 1, 1), (1, 9, 7, 1, 0, 0), (3, 50, 96, 12, 32, 0), (2, 40, 48, 4, 8, 3),
    (1, 1024, 64, 8, 0, 0), (2, 5000, 16, 4, 0, 0), (1, 65536, 8, 2, 0, 0), (1, 300, 1000, 10, 0, 0),
    (2, 20, 2304, 1, 0, 0), (300, 16, 128, 16, 0, 0), (2, 23296, 8, 2, 3, 0), (18, 900, 32, 4, 3, 1),
    (700, 5, 12, 3, 0, 0), (1, 30000, 136, 17, 0, 0), (2, 700, 272, 2, 0, 0), (3, 3500, 64, 8, 0, 0),
]


def _norm_case(shape, kind, act, seed, params=True):
    n, p, c, g, pad, shift = shape
    gen = _gen(seed)
    dtype, code = TYPES[kind]
    x, xbuf = _lay(_normal(gen, n, p, c, scale=1.5, mean=0.7), dtype, pad, shift)
    gamma = _normal(gen, c, scale=0.3, mean=1.0) if params else None
    beta = _normal(gen, c, scale=0.3) if params else None
    desc = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=code, activation=ACTS[act],
                            epsilon=1e-5, x_sample_stride=p * (c + pad), x_position_stride=c + pad,
                            y_sample_stride=p * (c + pad), y_position_stride=c + pad,
                            dx_sample_stride=p * (c + pad), dx_position_stride=c + pad)
    return gen, dtype, x, gamma, beta, desc


def _param64(gamma, beta, c):
    one = torch.ones(c, dtype=torch.float64, device="cuda")
    return (gamma.double() if gamma is not None else one), (beta.double() if beta is not None else 0 * one)


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_group_norm_forward(shape, kind):
    n, p, c, g, pad, shift = shape
    acts = list(ACTS)
    for act, params in ((acts[(n + p + c) % 4], True), ("silu", c % 2 == 0)):
        gen, dtype, x, gamma, beta, desc = _norm_case(shape, kind, act, 3, params)
        y, ybuf = _lay(torch.full((n, p, c), NAN, device="cuda"), dtype, pad, shift)
        mean, rstd = torch.full((2, n, g), NAN, device="cuda")
        work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
        assert tb.tb_cuda_group_norm_device(desc, x, gamma, beta, y, mean, rstd, work) == 1
        torch.cuda.synchronize()
        ga, be = _param64(gamma, beta, c)
        want = ref.group_norm(x.double(), ga, be, g, 1e-5, act)
        errs = ref.group_norm_errors(x.double(), ga, be, g, 1e-5, act)
        for name, got, w, e in zip(("y", "mean", "rstd"), (y, mean, rstd), want, errs):
            ref.check(f"{name} {act}", got, w, e)
        assert _untouched(y, ybuf, shift)
        again = y.clone()
        assert tb.tb_cuda_group_norm_device(desc, x, gamma, beta, y, None, None, work) == 1
        torch.cuda.synchronize()
        assert torch.equal(again, y)


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_group_norm_backward(shape, kind):
    n, p, c, g, pad, shift = shape
    acts = list(ACTS)
    for act, params in ((acts[(n + p + c + 1) % 4], True), ("silu", c % 2 == 0)):
        gen, dtype, x, gamma, beta, desc = _norm_case(shape, kind, act, 4, params)
        ga, be = _param64(gamma, beta, c)
        _, mean, rstd = (v.float() for v in ref.group_norm(x.double(), ga, be, g, 1e-5, act))
        if act == "relu":  # the slope jumps at 0: keep every u away from it
            hat = (x.double() - ref._wide(mean.double(), c // g)) * ref._wide(rstd.double(), c // g)
            close = (hat * ga + be).abs() < 1e-3
            x[close] += 0.05
        dy, _ = _lay(_normal(gen, n, p, c), dtype, pad, shift)
        dx, dxbuf = _lay(torch.full((n, p, c), NAN, device="cuda"), dtype, pad, shift)
        dgamma, dbeta = torch.full((2, c), NAN, device="cuda")
        work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
        assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta,
                                                     work) == 1
        torch.cuda.synchronize()
        want, errs = ref.group_norm_backward(x.double(), ga, be, mean.double(), rstd.double(), dy.double(), g, act)
        if act == "relu":
            hat = (x.double() - ref._wide(mean.double(), c // g)) * ref._wide(rstd.double(), c // g)
            if ((hat * ga + be).abs() < 1e-4).any():
                continue
        for name, got, w, e in zip(("dx", "dgamma", "dbeta"), (dx, dgamma, dbeta), want, errs):
            ref.check(f"{name} {act}", got, w, e)
        assert _untouched(dx, dxbuf, shift)
        first = [v.clone() for v in (dx, dgamma, dbeta)]
        assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta,
                                                     work) == 1
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, (dx, dgamma, dbeta)))
        # a dense dx from strided x and dy, and nothing written past it
        desc.dx_sample_stride = desc.dx_position_stride = 0
        dense, whole = _lay(torch.full((n, p, c), NAN, device="cuda"), dtype)
        assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, dy, dense, None, None, work) == 1
        torch.cuda.synchronize()
        ref.check(f"dense dx {act}", dense, want[0], errs[0])
        assert _untouched(dense, whole, 0)


def test_group_norm_in_place_and_partial_outputs():
    gen, dtype, x, gamma, beta, desc = _norm_case((3, 70, 64, 8, 0, 0), "bf16", "silu", 9)
    work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
    y, mean, rstd = torch.empty_like(x), torch.empty(3, 8, device="cuda"), torch.empty(3, 8, device="cuda")
    assert tb.tb_cuda_group_norm_device(desc, x, gamma, beta, y, mean, rstd, work) == 1
    dy = _normal(gen, 3, 70, 64).to(dtype)
    dx, dg, db = torch.empty_like(x), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, dy, dx, dg, db, work) == 1
    same, only = dy.clone(), torch.empty(64, device="cuda")
    assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, same, same, None, only, work) == 1
    over = x.clone()
    assert tb.tb_cuda_group_norm_backward_device(desc, over, gamma, beta, mean, rstd, dy, over, None, None, work) == 1
    x2 = x.clone()
    assert tb.tb_cuda_group_norm_device(desc, x2, gamma, beta, x2, None, None, work) == 1
    torch.cuda.synchronize()
    assert torch.equal(same, dx) and torch.equal(only, db) and torch.equal(over, dx) and torch.equal(x2, y)


def test_group_norm_large_mean_and_constant_groups():
    """A mean 1,000 deviations away loses nothing to cancellation, a constant group gives beta."""
    n, p, c, g = 2, 4096, 16, 2
    gen = _gen(5)
    x = _normal(gen, n, p, c) + 1000.0
    x[1, :, :8] = 7.25
    desc = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=0, activation=0, epsilon=1e-5)
    y, mean, rstd = torch.empty_like(x), torch.empty(n, g, device="cuda"), torch.empty(n, g, device="cuda")
    work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
    assert tb.tb_cuda_group_norm_device(desc, x, None, None, y, mean, rstd, work) == 1
    torch.cuda.synchronize()
    one = torch.ones(c, dtype=torch.float64, device="cuda")
    want = ref.group_norm(x.double(), one, 0 * one, g, 1e-5, "none")
    errs = ref.group_norm_errors(x.double(), one, 0 * one, g, 1e-5, "none")
    for name, got, w, e in zip(("y", "mean", "rstd"), (y, mean, rstd), want, errs):
        ref.check(name, got, w, e)
    assert float(y[1, :, :8].abs().max()) == 0.0


@pytest.mark.parametrize("kind", TYPES)
def test_group_norm_keeps_nan_in_its_group(kind):
    dtype, code = TYPES[kind]
    x = _normal(_gen(6), 3, 40, 32).to(dtype)
    x[1, 17, 9] = NAN
    x[2, 3, 30] = float("inf")
    desc = tb.GroupNormDesc(samples=3, positions=40, channels=32, groups=4, type=code, activation=2, epsilon=1e-5)
    y = torch.empty_like(x)
    work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
    assert tb.tb_cuda_group_norm_device(desc, x, None, None, y, None, None, work) == 1
    torch.cuda.synchronize()
    bad = torch.isnan(y).reshape(3, 40, 4, 8).any(3).any(1).cpu()
    assert bad.tolist() == [[False] * 4, [False, True, False, False], [False, False, False, True]]


# ---- gated recurrence ----

RECURRENCE_SHAPES = [
    # sequences, steps, channels, pad, shift
    (1, 1, 1, 0, 0), (3, 1, 64, 0, 0), (2, 2, 5, 0, 0), (2, 15, 33, 3, 1), (2, 16, 64, 0, 0), (1, 17, 130, 0, 0),
    (3, 100, 48, 16, 0), (2, 257, 64, 0, 0), (1, 1000, 96, 0, 0), (5, 129, 321, 0, 0), (1, 4099, 8, 0, 0),
    (40, 40, 256, 0, 0), (2, 333, 200, 8, 4),
    # tiles enough that one CTA takes many rounds: bulk copies
    (150, 260, 136, 0, 0), (600, 100, 72, 8, 0), (310, 300, 40, 8, 0),
    # few steps of many sequences
    (700, 1, 190, 0, 0), (64, 1, 512, 0, 0), (3000, 3, 128, 8, 0), (90, 8, 37, 2, 1),
    (5000, 2, 144, 0, 0), (40, 9, 64, 0, 0),
    (1300, 16, 128, 0, 0), (1200, 17, 32, 0, 0),
    # many rows, step by step
    (600, 50, 136, 0, 0), (300, 37, 131, 0, 0), (1700, 20, 512, 0, 0), (2400, 21, 33, 0, 0),
]


def _recurrence_case(shape, kind, resets, ragged, seed):
    b, t, d, pad, shift = shape
    gen = _gen(seed)
    dtype, code = TYPES[kind]
    s = {"dtype": dtype}
    xs, _ = _lay(_normal(gen, b, t, 3 * d), dtype, pad, shift)
    s["x"], s["rec"], s["inp"] = xs[..., :d], xs[..., d:2 * d], xs[..., 2 * d:]
    s["decay"] = _normal(gen, d, scale=1.5, mean=-2.0)
    s["state"] = _normal(gen, b, d)
    s["reset"] = (torch.rand((b, t), generator=gen, device="cuda") < 0.1).to(torch.uint8) * 255 if resets else None
    s["lengths"] = None
    if ragged:
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=gen, device="cuda").to(torch.int32)
        s["lengths"][0] = -3 if b > 2 else 0
        s["lengths"][-1] = t + 5
        past = torch.arange(t, device="cuda")[None] >= s["lengths"][:, None]
        xs[past] = NAN  # masked places may hold anything
    s["desc"] = tb.GatedRecurrenceDesc(
        sequences=b, steps=t, channels=d, type=code, decay_scale=8.0, in_sequence_stride=t * (3 * d + pad),
        in_step_stride=3 * d + pad, out_sequence_stride=t * (d + pad), out_step_stride=d + pad,
        grad_sequence_stride=t * (3 * d + pad), grad_step_stride=3 * d + pad)
    s["work"] = _scratch(tb.tb_cuda_gated_recurrence_workspace(s["desc"]))
    s["dh"], _ = _lay(_normal(gen, b, t, d), dtype, pad, shift)
    s["dstate"] = _normal(gen, b, d)
    if ragged:
        s["dh"][past] = NAN
    s["past"] = past if ragged else None
    return s


def _recurrence_reference(s, back):
    lengths = s["lengths"].clamp(min=0) if s["lengths"] is not None else None
    dh = s["dh"].double()
    if s["past"] is not None:
        dh = torch.where(s["past"][..., None], 0.0, dh)
    return ref.recurrence(s["x"].double(), s["rec"].double(), s["inp"].double(), s["decay"].double(), 8.0, s["reset"],
                          lengths, s["state"].double(), dh if back else None, s["dstate"].double())


@pytest.mark.parametrize("shape", RECURRENCE_SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_gated_recurrence(shape, kind):
    b, t, d, pad, shift = shape
    for seed, (resets, ragged) in enumerate(itertools.product((False, True), repeat=2)):
        s = _recurrence_case(shape, kind, resets, ragged, seed + 20)
        want = _recurrence_reference(s, True)
        h, hbuf = _lay(torch.full((b, t, d), NAN, device="cuda"), s["dtype"], pad, shift)
        out = torch.full((b, d), NAN, device="cuda")
        saved = torch.full((b, -(-t // 16), d), NAN, device="cuda")
        args = (s["desc"], s["x"], s["rec"], s["inp"], s["decay"], s["reset"], s["lengths"], s["state"])
        assert tb.tb_cuda_gated_recurrence_device(*args, h, out, saved, s["work"]) == 1
        torch.cuda.synchronize()
        for name, got in (("h", h), ("state", out), ("checkpoints", saved)):
            ref.check(name, got, *want[name])
        assert _untouched(h, hbuf, shift)
        h2, again = h.clone(), out.clone()
        assert tb.tb_cuda_gated_recurrence_device(*args, h, out, None, s["work"]) == 1
        torch.cuda.synchronize()
        assert torch.equal(h2, h) and torch.equal(again, out)

        grads, gbuf = _lay(torch.full((b, t, 3 * d), NAN, device="cuda"), s["dtype"], pad, shift)
        dx, drec, dinp = grads[..., :d], grads[..., d:2 * d], grads[..., 2 * d:]
        ddecay, dstate = torch.full((d,), NAN, device="cuda"), torch.full((b, d), NAN, device="cuda")
        back = args[:7] + (saved, s["dh"], s["dstate"], dx, drec, dinp, ddecay, dstate, s["work"])
        assert tb.tb_cuda_gated_recurrence_backward_device(*back) == 1
        torch.cuda.synchronize()
        for name, got in (("dx", dx), ("drec", drec), ("dinp", dinp), ("ddecay", ddecay), ("dstate", dstate)):
            ref.check(name, got, *want[name])
        assert _untouched(grads, gbuf, shift)
        first = [v.clone() for v in (grads, ddecay, dstate)]
        assert tb.tb_cuda_gated_recurrence_backward_device(*back) == 1
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(first, (grads, ddecay, dstate)))


def test_gated_recurrence_steps_in_place_like_one_scan():
    """Acting one step at a time with the state in place gives the bits of the state of a whole scan, reset by reset."""
    s = _recurrence_case((4, 37, 70, 0, 0), "bf16", True, False, 3)
    h = torch.empty((4, 37, 70), dtype=torch.bfloat16, device="cuda")
    out = torch.empty((4, 70), device="cuda")
    desc = tb.GatedRecurrenceDesc(sequences=4, steps=37, channels=70, type=1, decay_scale=8.0,
                                  in_sequence_stride=37 * 210, in_step_stride=210)
    assert tb.tb_cuda_gated_recurrence_device(desc, s["x"], s["rec"], s["inp"], s["decay"], s["reset"], None,
                                              s["state"], h, out, None, s["work"]) == 1
    step = tb.GatedRecurrenceDesc(sequences=4, steps=1, channels=70, type=1, decay_scale=8.0,
                                  in_sequence_stride=37 * 210, in_step_stride=210)
    state, one = s["state"].clone(), torch.empty((4, 1, 70), dtype=torch.bfloat16, device="cuda")
    work = _scratch(tb.tb_cuda_gated_recurrence_workspace(step))
    for t in range(37):
        flags = s["reset"][:, t].contiguous()
        assert tb.tb_cuda_gated_recurrence_device(step, s["x"][:, t:], s["rec"][:, t:], s["inp"][:, t:], s["decay"],
                                                  flags, None, state, one, state, None, work) == 1
    torch.cuda.synchronize()
    want = _recurrence_reference(s, False)
    ref.check("state", state, *want["state"])
    ref.check("state of the scan", out, *want["state"])


def test_gated_recurrence_null_states_and_extreme_gates():
    """NULL states are zeros; shut and open gates, a decay of nothing and of all, give finite gradients."""
    b, t, d = 2, 50, 40
    s = _recurrence_case((b, t, d, 0, 0), "f32", False, False, 8)
    s["rec"][:, ::3] = 200.0
    s["rec"][:, 1::3] = -200.0
    s["inp"][:, ::5] = -150.0
    s["decay"][:10], s["decay"][10:20] = -300.0, 90.0
    s["state"], s["dstate"] = torch.zeros(b, d, device="cuda"), torch.zeros(b, d, device="cuda")
    want = _recurrence_reference(s, True)
    h, saved = torch.empty((b, t, d), device="cuda"), torch.empty((b, 4, d), device="cuda")
    assert tb.tb_cuda_gated_recurrence_device(s["desc"], s["x"], s["rec"], s["inp"], s["decay"], None, None, None, h,
                                              None, saved, s["work"]) == 1
    grads = torch.empty((b, t, 3 * d), device="cuda")
    dx, drec, dinp = grads[..., :d], grads[..., d:2 * d], grads[..., 2 * d:]
    ddecay = torch.empty(d, device="cuda")
    assert tb.tb_cuda_gated_recurrence_backward_device(
        s["desc"], s["x"], s["rec"], s["inp"], s["decay"], None, None, saved, s["dh"], None, dx, drec, dinp, ddecay,
        None, s["work"]) == 1
    torch.cuda.synchronize()
    # below f32's smallest normal numbers a product may be flushed: allow it 2^-126 of a magnitude of at most 1e6
    for name, got in (("h", h), ("dx", dx), ("drec", drec), ("dinp", dinp), ("ddecay", ddecay)):
        assert torch.isfinite(got).all(), name
        value, bound = want[name]
        ref.check(name, got, value, bound + 1e-30)


# ---- routing ----

ROUTE_CASES = [
    # tokens, experts, top_k, groups, top_groups, group_best, score, bias, renormalise
    (1, 1, 1, 1, 1, 1, "softmax", False, True), (5, 3, 3, 1, 1, 1, "sigmoid", False, False),
    (33, 8, 2, 1, 1, 1, "softmax", False, True), (70, 60, 6, 1, 1, 1, "softmax", False, False),
    (61, 64, 6, 8, 3, 2, "sigmoid", True, True), (50, 64, 8, 4, 2, 1, "softmax", False, True),
    (40, 256, 8, 8, 4, 2, "sigmoid", True, True), (20, 257, 4, 1, 1, 1, "sigmoid", True, False),
    (30, 96, 5, 3, 2, 2, "sigmoid", False, True), (12, 1024, 32, 1, 1, 1, "softmax", False, True),
    (300, 16, 16, 1, 1, 1, "softmax", True, False), (9, 512, 12, 16, 5, 2, "softmax", True, True),
    (25, 40, 7, 40, 9, 2, "sigmoid", True, True), (6, 1000, 3, 500, 2, 1, "sigmoid", False, False),
    (500, 12, 4, 1, 1, 1, "sigmoid", True, True), (17, 130, 9, 2, 1, 2, "sigmoid", True, True),
]


def _route_desc(case, code, stride=0, scale=1.0):
    t, e, k, g, tg, gb, score, _, renorm = case
    return tb.ExpertRouteDesc(tokens=t, experts=e, top_k=k, groups=g, top_groups=tg, group_best=gb, type=code,
                              score=tb.TB_SCORE_SOFTMAX if score == "softmax" else tb.TB_SCORE_SIGMOID,
                              renormalise=int(renorm), weight_scale=scale, logits_stride=stride)


def _route(desc, logits, bias, t, e, k, lists=True):
    new = lambda *s: torch.full(s, -77, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, weights = new(t, k), torch.full((t, k), NAN, device="cuda")
    more = (new(e + 1), new(t * k), new(t, k)) if lists else (None, None, None)
    work = _scratch(tb.tb_cuda_route_experts_workspace(desc))
    assert tb.tb_cuda_route_experts_device(desc, logits, bias, ids, weights, *more, work) == 1
    torch.cuda.synchronize()
    return (ids, weights) + more


def _route_logits(case, kind, seed, masks):
    t, e = case[:2]
    gen = _gen(seed)
    logits = _normal(gen, t, e, scale=2.0)
    if masks:
        logits[torch.rand((t, e), generator=gen, device="cuda") < 0.3] = float("-inf")
        logits[::7] = float("-inf")               # nothing is available
        logits[3::11, e // 2] = NAN               # not available either
        logits[5::13, :max(1, e // 3)] = 1.25     # ties
        logits[1::17, 0] = torch.finfo(torch.float32).min if kind != "f16" else torch.finfo(torch.float16).min
    bias = torch.randint(-30, 31, (e,), generator=gen, device="cuda") * 0.01 if case[7] else None
    return logits.to(TYPES[kind][0]), bias


@pytest.mark.parametrize("case", ROUTE_CASES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("masks", (False, True))
def test_route_experts(case, kind, masks):
    t, e, k, g, tg, gb, score, _, renorm = case
    logits, bias = _route_logits(case, kind, 31, masks)
    wide = torch.full((t, e + 5), NAN, dtype=logits.dtype, device="cuda")
    wide[:, 2:e + 2] = logits
    ids, weights, offsets, order, position = _route(_route_desc(case, TYPES[kind][1], e + 5, 1.5), wide[:, 2:], bias,
                                                    t, e, k)
    want, w64, gap = ref.route(logits.cpu(), bias.cpu() if bias is not None else None, score, k, g, tg, gb, renorm, 1.5)
    # rankings are stated in f32: tokens whose 64-bit ranking values lie within a few roundings are not compared
    clear = gap > 16 * ref.U * 2
    if bias is None and not (g > 1 and gb == 2):
        clear[:] = True
    else:
        assert masks or clear.float().mean() > 0.9
        for r in torch.nonzero(~clear).flatten().tolist():  # still: distinct, available, best first
            got = [i for i in ids[r].tolist() if i >= 0]
            assert len(set(got)) == len(got) == int((want[r] >= 0).sum())
            want[r] = ids[r].cpu()
    assert torch.equal(ids.cpu().long()[clear], want[clear])
    same = ref.route_weights(ref.available(logits.double().cpu()), ids.cpu().long(), score, renorm, 1.5)
    # scores within 8 U and (softmax) |logit spread| U of the exponent; sums of at most 1024 terms; one division
    spread = ref.available(logits.double().cpu())
    spread = torch.where(torch.isfinite(spread), spread, 0.0).abs().amax(1, keepdim=True).clamp(max=200)
    ref.check("weights", weights, same.to("cuda"), ((64 + 4 * spread) * ref.U * same).to("cuda") + 1e-37)
    # the lists follow from the ids
    o, lst, pos = ref.slot_lists(ids.cpu(), e)
    assert offsets.tolist() == o and order.tolist() == lst and position.flatten().tolist() == pos
    only = _route(_route_desc(case, TYPES[kind][1], e + 5, 1.5), wide[:, 2:], bias, t, e, k, lists=False)
    assert torch.equal(only[0], ids) and torch.equal(only[1], weights)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 8, 2), (127, 4, 2), (128, 4, 2), (129, 256, 8), (5000, 64, 6),
                                                  (40001, 24, 3), (70000, 300, 2)])
def test_route_slot_lists_at_scale(tokens, experts, top_k):
    """Lists over many tiles, with tokens without experts and an expert that takes nearly all."""
    gen = _gen(12)
    logits = _normal(gen, tokens, experts)
    logits[:, 1] += 6.0
    logits[torch.rand((tokens,), generator=gen, device="cuda") < 0.2] = float("-inf")
    case = (tokens, experts, top_k, 1, 1, 1, "softmax", False, True)
    ids, weights, offsets, order, position = _route(_route_desc(case, 0), logits, None, tokens, experts, top_k)
    want = logits.sort(dim=1, descending=True, stable=True)[1][:, :top_k]
    want = torch.where(torch.isinf(logits).all(1)[:, None], -1, want)
    assert torch.equal(ids.long(), want)
    key = torch.where(ids.flatten() >= 0, ids.flatten(), experts).long()
    skey, perm = key.sort(stable=True)
    assert torch.equal(offsets.long(), torch.searchsorted(skey, torch.arange(experts + 1, device="cuda")))
    assert torch.equal(order.long(), torch.where(skey < experts, perm, -1))
    place = torch.full_like(key, -1)
    place[perm[skey < experts]] = torch.arange(int((skey < experts).sum()), device="cuda")
    assert torch.equal(position.flatten().long(), place)


def test_route_infinite_logits():
    logits = torch.tensor([[float("inf"), 0.0, float("inf"), 1.0], [float("-inf"), NAN, 2.0, float("-inf")]],
                          device="cuda")
    ids, weights, *_ = _route(_route_desc((2, 4, 3, 1, 1, 1, "softmax", False, False), 0), logits, None, 2, 4, 3)
    assert ids.tolist() == [[0, 2, 3], [2, -1, -1]]
    assert weights.tolist() == [[0.5, 0.5, 0.0], [1.0, 0.0, 0.0]]


@pytest.mark.parametrize("case", ROUTE_CASES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_route_backward(case, kind):
    t, e, k, g, tg, gb, score, _, renorm = case
    dtype, code = TYPES[kind]
    logits, bias = _route_logits(case, kind, 33, True)
    ids, _, _ = ref.route(logits.cpu(), bias.cpu() if bias is not None else None, score, k, g, tg, gb, renorm, 1.5)
    gen = _gen(34)
    dw = _normal(gen, t, k)
    dlogits, buf = _lay(torch.full((1, t, e), NAN, device="cuda"), dtype, 5, 2)
    wide = torch.full((t, e + 5), NAN, dtype=dtype, device="cuda")
    wide[:, :e] = logits
    desc = _route_desc(case, code, e + 5, 1.5)
    assert tb.tb_cuda_route_experts_backward_device(desc, wide, ids.to("cuda", torch.int32), dw, dlogits) == 1
    torch.cuda.synchronize()
    l64 = ref.available(logits.double().cpu())
    l64 = torch.where(torch.isneginf(l64), -1e300, l64).requires_grad_(True)
    w = ref.route_weights(l64, ids, score, renorm, 1.5)
    want = torch.autograd.grad(w, l64, dw.double().cpu())[0]
    want = torch.where(ref.available(logits.double().cpu()) > float("-inf"), want, 0.0)
    # each score within (16 + 4 spread) U; a slot's gradient is a difference of terms of at most
    # |dw_j| + the weighted mean of |dw|, over the sum of the scores where they are renormalised
    s = ref.scores(l64.detach(), score)
    pick = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0)), 0.0)
    total = pick.sum(1, keepdim=True).clamp(min=1e-300) if renorm else torch.ones((t, 1), dtype=torch.float64)
    top = 1.5 * torch.where(ids >= 0, dw.double().cpu().abs(), 0.0)
    size = torch.zeros_like(s).scatter_add_(1, ids.clamp(min=0), (top + renorm * (top * pick).sum(1, keepdim=True) / total) / total)
    if score == "softmax":
        size = size + (size * s).sum(1, keepdim=True)
    spread = torch.where(l64.detach() > -1e299, l64.detach(), 0.0).abs().amax(1, keepdim=True).clamp(max=200)
    bound = (96 + 8 * spread) * ref.U * s * size
    ref.check("dlogits", dlogits[0], want.to("cuda"), bound.to("cuda") + 1e-37)
    assert _untouched(dlogits, buf, 2)


# ---- combine ----

COMBINE_SHAPES = [(1, 1, 1, 0, 0), (7, 2, 33, 0, 0), (61, 6, 520, 0, 0), (40, 8, 128, 8, 0), (30, 3, 264, 8, 4),
                  (5, 32, 1000, 0, 0), (300, 4, 72, 3, 1), (20, 1, 4096, 0, 0), (10, 12, 2049, 0, 0),
                  (50, 3, 36, 0, 0), (50, 5, 66, 8, 2)]


@pytest.mark.parametrize("shape", COMBINE_SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("weighted", (True, False))
def test_combine(shape, kind, weighted):
    t, k, w, pad, shift = shape
    dtype, code = TYPES[kind]
    gen = _gen(41)
    r = t * k + 3
    rows, _ = _lay(_normal(gen, 1, r, w), dtype, pad, shift)
    position = torch.randperm(r, generator=gen, device="cuda")[:t * k].reshape(t, k).to(torch.int32)
    position[torch.rand((t, k), generator=gen, device="cuda") < 0.2] = -1
    position[0] = -1                       # a token without any expert
    if t > 2:
        position[2, 0] = r + 4             # outside the rows: adds nothing
    weights = _normal(gen, t, k) if weighted else None
    out, obuf = _lay(torch.full((1, t, w), NAN, device="cuda"), dtype, pad, shift)
    desc = tb.ExpertCombineDesc(tokens=t, rows=r, width=w, top_k=k, type=code, rows_stride=w + pad, out_stride=w + pad)
    there = (position >= 0) & (position < r)
    named = torch.zeros(r, dtype=torch.bool, device="cuda")
    named[position[there].long()] = True
    rows[0][~named] = NAN  # rows that none names may hold anything
    assert tb.tb_cuda_combine_experts_device(desc, rows, position, weights, out) == 1
    torch.cuda.synchronize()
    w64 = torch.where(there, weights.double() if weighted else 1.0, 0.0)[..., None]
    picked = torch.where(there[..., None], rows[0].double()[torch.where(there, position, 0).long()], 0.0)
    want = (picked * w64).sum(1)
    ref.check("out", out[0], want, (k + 2) * ref.U * (picked * w64).abs().sum(1))
    assert _untouched(out, obuf, shift)

    dout, _ = _lay(_normal(gen, 1, t, w), dtype, pad, shift)
    drows, dbuf = _lay(torch.full((1, r, w), NAN, device="cuda"), dtype, pad, shift)
    dweights = torch.full((t, k), NAN, device="cuda")
    assert tb.tb_cuda_combine_experts_backward_device(desc, rows, position, weights, dout, drows, dweights) == 1
    torch.cuda.synchronize()
    prod = dout[0].double()[:, None] * picked
    # a dot product in partial sums of at most w/32 terms, then log2
    ref.check("dweights", dweights, prod.sum(2), (w / 32 + 16) * ref.U * prod.abs().sum(2))
    d64 = (w64 if weighted else there[..., None].double()) * dout[0].double()[:, None]
    ref.check("drows", drows[0][position[there].long()], d64[there], 2 * ref.U * d64[there].abs())
    assert torch.isnan(drows[0][~named]).all() and _untouched(drows, dbuf, shift)
    only = torch.full_like(drows, NAN)
    dense = tb.ExpertCombineDesc(tokens=t, rows=r, width=w, top_k=k, type=code, out_stride=w + pad)
    assert tb.tb_cuda_combine_experts_backward_device(dense, None, position, weights, dout, only, None) == 1
    torch.cuda.synchronize()
    assert torch.equal(only[0][named], drows[0][named])


# ---- streams ----

def test_calls_follow_their_stream():
    """Work queued behind a long wait on a side stream sees the inputs written there, not those of another stream."""
    side = torch.cuda.Stream()
    n, p, c, g = 4, 64, 64, 8
    x, y = torch.zeros((n, p, c), device="cuda"), torch.empty((n, p, c), device="cuda")
    new = _normal(_gen(1), n, p, c)
    desc = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=0, activation=2, epsilon=1e-5)
    work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
    want = torch.empty_like(y)
    assert tb.tb_cuda_group_norm_device(desc, new, None, None, want, None, None, work) == 1
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x.copy_(new)
        assert tb.tb_cuda_group_norm_device(desc, x, None, None, y, None, None, work, side) == 1
    side.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("shape,kind", [((3, 3001, 321), "f32"), ((2, 257, 64), "bf16"), ((8, 1000, 512), "bf16"),
                                        ((1, 4099, 40), "f16"), ((5, 700, 96), "f32"), ((4, 5, 24), "f32")], ids=str)
@pytest.mark.parametrize("busy", (False, True))
def test_gated_recurrence_in_place_over_many_steps(shape, kind, busy):
    """state_out on state_in, and dstate_in on dstate_out, give the bits of separate buffers, also where the steps are
    cut into strips and other work holds up some of them."""
    b, t, d = shape
    s = _recurrence_case((b, t, d, 0, 0), kind, True, True, 13)
    new = lambda *n, dtype=torch.float32: torch.full(n, NAN, dtype=dtype, device="cuda")  # noqa: E731
    args = (s["desc"], s["x"], s["rec"], s["inp"], s["decay"], s["reset"], s["lengths"])
    other, m = torch.cuda.Stream(), torch.ones((2048, 2048), device="cuda")

    def run(in_place):
        out, dout = new(b, d), new(b, d)
        first, last = s["state"], s["dstate"]
        if in_place:
            first, last = out, dout = s["state"].clone(), s["dstate"].clone()
        h, saved = new(b, t, d, dtype=s["dtype"]), new(b, -(-t // 16), d)
        grads, ddecay = new(b, t, 3 * d, dtype=s["dtype"]), new(d)
        torch.cuda.synchronize()
        if busy:
            with torch.cuda.stream(other):
                for _ in range(4):
                    m @ m
        assert tb.tb_cuda_gated_recurrence_device(*args, first, h, out, saved, s["work"]) == 1
        assert tb.tb_cuda_gated_recurrence_backward_device(*args, saved, s["dh"], last, grads, grads[..., d:],
                                                           grads[..., 2 * d:], ddecay, dout, s["work"]) == 1
        torch.cuda.synchronize()
        return h, saved, grads, ddecay, out, dout

    want = run(False)
    for _ in range(4):
        assert all(torch.equal(a, c) for a, c in zip(want, run(True)))
    if not busy:
        exact = _recurrence_reference(s, True)
        for name, got in (("state", want[4]), ("dstate", want[5])):
            ref.check(name, got, *exact[name])


RESET_SHAPES = [(2, 15, 33), (3, 100, 48), (2, 257, 64), (1, 1000, 96), (5, 129, 321), (8, 1000, 128), (150, 260, 136),
                (310, 300, 40), (64, 1, 512), (90, 8, 37), (600, 50, 136), (700, 1, 190)]


def _recurrence_run(s, shape, state, dh, dstate):
    """Every output of both directions, the backward pass from the forward pass's checkpoints."""
    b, t, d = shape
    new = lambda *n, dtype=torch.float32: torch.full(n, 7.0, dtype=dtype, device="cuda")  # noqa: E731
    o = {"h": new(b, t, d, dtype=s["dtype"]), "state": new(b, d), "checkpoints": new(b, -(-t // 16), d),
         "grads": new(b, t, 3 * d, dtype=s["dtype"]), "ddecay": new(d), "dstate": new(b, d)}
    args = (s["desc"], s["x"], s["rec"], s["inp"], s["decay"], s["reset"], s["lengths"])
    assert tb.tb_cuda_gated_recurrence_device(*args, state, o["h"], o["state"], o["checkpoints"], s["work"]) == 1
    assert tb.tb_cuda_gated_recurrence_backward_device(
        *args, o["checkpoints"], dh, dstate, o["grads"], o["grads"][..., d:], o["grads"][..., 2 * d:], o["ddecay"],
        o["dstate"], s["work"]) == 1
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("shape", RESET_SHAPES, ids=str)
@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_gated_recurrence_starts_anew_from_any_state(shape, kind):
    """An episode's first step forgets a state that nobody set: with a reset at step 0, states of NaN and infinities
    give the bits that zeros give, forward and backward."""
    b, t, d = shape
    s = _recurrence_case((b, t, d, 0, 0), kind, True, False, 51)
    s["reset"][:, 0] = 1
    want = _recurrence_run(s, shape, torch.zeros((b, d), device="cuda"), s["dh"], s["dstate"])
    state = torch.full((b, d), NAN, device="cuda")
    state[:, 1::3] = float("inf")
    state[:, 2::3] = -float("inf")
    got = _recurrence_run(s, shape, state, s["dh"], s["dstate"])
    assert torch.equal(got["checkpoints"][:, 1:], want["checkpoints"][:, 1:])
    for name in ("h", "state", "grads", "ddecay", "dstate"):
        assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("shape", [n for n in RESET_SHAPES if n[1] > 8], ids=str)
@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_gated_recurrence_keeps_episodes_apart(shape, kind):
    """NaN inputs of an episode's last step reach its state and no later step, and a NaN gradient of the last state no
    place past a sequence's length."""
    b, t, d = shape
    s = _recurrence_case((b, t, d, 0, 0), kind, True, False, 52)
    turn = torch.randint(2, t, (b,), generator=_gen(53), device="cuda")  # an episode's first step
    row = torch.arange(b, device="cuda")
    s["reset"][row, turn], s["reset"][row, turn - 1] = 1, 0
    want = _recurrence_run(s, shape, s["state"], s["dh"], s["dstate"])
    step = torch.arange(t, device="cuda")[None]
    later, last = step >= turn[:, None], step == turn[:, None] - 1
    clean = [s[name].clone() for name in ("x", "rec", "inp")]
    for i, name in enumerate(("x", "rec", "inp")):  # a third of the channels each
        s[name][..., i::3] = torch.where(last[..., None], NAN, s[name][..., i::3])
    got = _recurrence_run(s, shape, s["state"], s["dh"], s["dstate"])
    assert torch.isnan(got["h"][last]).all()
    assert torch.equal(got["h"][later], want["h"][later]) and torch.equal(got["state"], want["state"])
    saved = torch.arange(0, t, 16, device="cuda")[None] > turn[:, None]  # the state before the step
    assert torch.equal(got["checkpoints"][saved], want["checkpoints"][saved])
    for v, name in zip(clean, ("x", "rec", "inp")):
        s[name].copy_(v)
    s["lengths"] = turn.to(torch.int32)
    got = _recurrence_run(s, shape, s["state"], s["dh"], torch.full((b, d), NAN, device="cuda"))
    assert float(got["grads"][later].abs().max()) == 0.0 and float(got["h"][later].abs().max()) == 0.0


@pytest.mark.parametrize("shape", RESET_SHAPES, ids=str)
@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_gated_recurrence_of_empty_sequences(shape, kind):
    """Sequences of length 0 hand their state on, NaN too, and leave no trace in the gradients."""
    b, t, d = shape
    s = _recurrence_case((b + 1, t, d, 0, 0), kind, False, False, 54)
    shape = (b + 1, t, d)
    s["lengths"] = torch.full((b + 1,), t, dtype=torch.int32, device="cuda")
    s["lengths"][b // 2] = 0
    want = _recurrence_run(s, shape, s["state"], s["dh"], s["dstate"])
    state = s["state"].clone()
    state[b // 2] = NAN
    for name in ("x", "rec", "inp"):
        s[name][b // 2] = float("inf")
    got = _recurrence_run(s, shape, state, s["dh"], s["dstate"])
    assert torch.isnan(got["state"][b // 2]).all() and float(got["h"][b // 2].abs().max()) == 0.0
    for name in ("grads", "ddecay", "dstate"):
        assert torch.equal(got[name], want[name]), name
    assert torch.equal(got["dstate"][b // 2], s["dstate"][b // 2])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", [(1, 20000, 272, 1, 3), (2, 9000, 1300, 2, 1), (1, 700, 2304, 1, 0),
                                   (5, 1, 2304, 1, 0), (6, 3, 1300, 2, 1), (2, 7, 4100, 4, 0), (2, 15, 5000, 2, 0)], ids=str)
def test_group_norm_of_wide_groups_and_many_positions(shape, kind):
    """Groups wider than a CTA's rows: hundreds of thousands of values a thread, of one sign and nearly one size, cost
    no more digits than the bounds allow."""
    n, p, c, g, pad = shape
    dtype, code = TYPES[kind]
    gen = _gen(61)
    x, _ = _lay(_normal(gen, n, p, c) + 1003.0, dtype, pad)
    y, ybuf = _lay(torch.full((n, p, c), NAN, device="cuda"), dtype, pad)
    desc = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=code, activation=ACTS["none"],
                            epsilon=1e-5, x_sample_stride=p * (c + pad), x_position_stride=c + pad,
                            y_sample_stride=p * (c + pad), y_position_stride=c + pad)
    mean, rstd = torch.full((2, n, g), NAN, device="cuda")
    work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
    assert tb.tb_cuda_group_norm_device(desc, x, None, None, y, mean, rstd, work) == 1
    torch.cuda.synchronize()
    ga, be = _param64(None, None, c)
    want = ref.group_norm(x.double(), ga, be, g, 1e-5, "none")
    errs = ref.group_norm_errors(x.double(), ga, be, g, 1e-5, "none")
    for name, got, w, e in zip(("y", "mean", "rstd"), (y, mean, rstd), want, errs):
        ref.check(name, got, w, e)
    assert _untouched(y, ybuf, 0)
    mean, rstd = want[1].float(), want[2].float()
    del want, errs, y, ybuf
    dy, _ = _lay(_normal(gen, n, p, c) * 0.01 + 1.003, dtype, pad)
    dx = torch.full((n, p, c), NAN, dtype=dtype, device="cuda")
    dgamma, dbeta = torch.full((2, c), NAN, device="cuda")
    assert tb.tb_cuda_group_norm_backward_device(desc, x, None, None, mean, rstd, dy, dx, dgamma, dbeta, work) == 1
    torch.cuda.synchronize()
    want, errs = ref.group_norm_backward(x.double(), ga, be, mean.double(), rstd.double(), dy.double(), g, "none")
    for name, got, w, e in zip(("dx", "dgamma", "dbeta"), (dx, dgamma, dbeta), want, errs):
        ref.check(name, got, w, e)


@pytest.mark.parametrize("shape", [(2, 50, 40), (3, 1, 40), (2, 700, 40), (200, 40, 40)], ids=str)
def test_gated_recurrence_of_infinite_decays(shape):
    """A decay of +inf or near f32's highest forgets every state, one of -inf or near the lowest keeps it; NaN is
    NaN, in its channel.  No gradient of the others is anything but finite."""
    b, t, d = shape
    s = _recurrence_case((b, t, d, 0, 0), "f32", True, False, 71)
    ends = torch.tensor([float("inf"), 3.4e38, 1e33, -float("inf"), -3.4e38, -1e33], device="cuda")
    s["decay"][:30] = ends.repeat(5)
    s["decay"][39] = NAN
    s["rec"].clamp_(min=-5.0)  # gates that are open at all
    o = _recurrence_run(s, shape, s["state"], s["dh"], s["dstate"])
    s["decay"][:30] = s["decay"][:30].clamp(-1e4, 1e4)  # as good as infinite: a is 0 or 1 in 64 bits too
    want = _recurrence_reference(s, True)
    keep = torch.arange(d, device="cuda") != 39
    got = dict(o, dx=o["grads"][..., :d], drec=o["grads"][..., d:2 * d], dinp=o["grads"][..., 2 * d:])
    for name in ("h", "state", "checkpoints", "dx", "drec", "dinp", "ddecay", "dstate"):
        value, bound = want[name]
        assert torch.isfinite(got[name][..., keep]).all(), name
        ref.check(name, got[name][..., keep], value[..., keep], bound[..., keep] + 1e-30)
    assert torch.isnan(o["ddecay"][39])


@pytest.mark.parametrize("top_k", (1, 2, 5, 16))
def test_route_renormalises_scores_near_the_smallest(top_k):
    """Sigmoid scores down to f32's last powers of two, all of a token's alike far down: their weights are ratios of
    order 1, and so are the gradients."""
    t, e = 400, 24
    gen = _gen(81)
    logits = -88.6 + 1.5 * torch.rand((t, e), generator=gen, device="cuda")
    logits[::3] += torch.rand((len(logits[::3]), 1), generator=gen, device="cuda") * 10
    desc = _route_desc((t, e, top_k, 1, 1, 1, "sigmoid", False, True), 0, 0, 1.0)
    ids, weights, *_ = _route(desc, logits, None, t, e, top_k)
    l64 = logits.double().cpu().requires_grad_(True)
    want, _, _ = ref.route(l64.detach(), None, "sigmoid", top_k, renormalise=True)
    assert torch.equal(ids.cpu().long(), want)
    w = ref.route_weights(l64, want, "sigmoid", True, 1.0)
    # each score within 8 U, and as it may be below the normal numbers, 2^-150 of at least 2.9e-39: 4 U; then sums and a division
    ref.check("weights", weights, w.detach().cuda(), 64 * ref.U * w.detach().cuda())
    dw = _normal(gen, t, top_k)
    dlogits = torch.full((t, e), NAN, device="cuda")
    assert tb.tb_cuda_route_experts_backward_device(desc, logits, ids, dw, dlogits) == 1
    torch.cuda.synchronize()
    grad = torch.autograd.grad(w, l64, dw.double().cpu())[0].cuda()
    size = torch.zeros((t, e), dtype=torch.float64, device="cuda")
    w64, top = w.detach().cuda(), dw.double().abs()
    size.scatter_add_(1, ids.long(), w64 * (top + (top * w64).sum(1, keepdim=True)))
    ref.check("dlogits", dlogits, grad, 96 * ref.U * size)


@pytest.mark.parametrize("shape", [(6, 1, 72), (3, 100, 48), (5, 129, 321), (150, 100, 136), (310, 130, 40),
                                   (600, 50, 136), (8, 700, 128)], ids=str)
@pytest.mark.parametrize("order", ("steps first", "gaps", "steps first, rows apart"))
@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_gated_recurrence_in_other_orders(shape, order, kind):
    """Tensors with the steps outermost, sequences at a distance that is no whole number of steps, and steps outermost of
    which each row is followed by a gap agree with the definition as dense ones do."""
    b, t, d = shape
    s = _recurrence_case((b, t, d, 0, 0), kind, True, True, 91)
    dtype = s["dtype"]
    wide = {"steps first": (d, b * d + 16), "gaps": (t * d + 24, d), "steps first, rows apart": (d + 8, b * (d + 8))}[order]
    dense = tb.GatedRecurrenceDesc(sequences=b, steps=t, channels=d, type=TYPES[kind][1], decay_scale=8.0)
    laid = tb.GatedRecurrenceDesc(
        sequences=b, steps=t, channels=d, type=TYPES[kind][1], decay_scale=8.0, in_sequence_stride=wide[0],
        in_step_stride=wide[1], out_sequence_stride=wide[0], out_step_stride=wide[1], grad_sequence_stride=wide[0],
        grad_step_stride=wide[1])
    size = (b - 1) * wide[0] + (t - 1) * wide[1] + d

    def lay(v):
        whole = torch.full((size + 8,), NAN, dtype=dtype, device="cuda")
        view = whole.as_strided((b, t, d), (*wide, 1))
        if v is not None:
            view.copy_(v)
        return view, whole

    def run(desc, place):
        x, rec, inp, dh = (place(s[n])[0] for n in ("x", "rec", "inp", "dh"))
        (h, hw), *grads = (place(None) for _ in range(4))
        out, dstate = torch.full((2, b, d), NAN, device="cuda")
        saved, ddecay = torch.full((b, -(-t // 16), d), NAN, device="cuda"), torch.full((d,), NAN, device="cuda")
        args = (desc, x, rec, inp, s["decay"], s["reset"], s["lengths"])
        assert tb.tb_cuda_gated_recurrence_device(*args, s["state"], h, out, saved, s["work"]) == 1
        assert tb.tb_cuda_gated_recurrence_backward_device(*args, saved, dh, s["dstate"], *(g for g, _ in grads), ddecay,
                                                           dstate, s["work"]) == 1
        torch.cuda.synchronize()
        return [h, *(g for g, _ in grads), out, saved, ddecay, dstate], [hw, *(w for _, w in grads)]

    want, _ = run(dense, lambda v: (v.contiguous() if v is not None else torch.empty((b, t, d), dtype=dtype, device="cuda"), None))
    got, wholes = run(laid, lay)
    exact = _recurrence_reference(s, True)
    for name, g, w in zip(("h", "dx", "drec", "dinp", "state", "checkpoints", "ddecay", "dstate"), got, want):
        ref.check(name, g, *exact[name])
        ref.check(name, w, *exact[name])
    for g, whole in zip(got, wholes):  # nothing between the rows is written
        assert int(torch.isnan(whole).sum()) == whole.numel() - g.numel()


@pytest.mark.parametrize("shape", [(3, 70, 1300, 1), (2, 5, 2304, 1), (1, 30000, 64, 8), (2, 3000, 64, 8), (40, 3, 12, 3)],
                         ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_group_norm_in_place_in_every_form(shape, kind):
    """y over x, dx over dy and dx over x give the bits of buffers of their own, whichever kernels the shape takes."""
    n, p, c, g = shape
    gen, dtype, x, gamma, beta, desc = _norm_case((n, p, c, g, 0, 0), kind, "gelu", 95)
    work = _scratch(tb.tb_cuda_group_norm_workspace(desc))
    y, mean, rstd = torch.empty_like(x), *torch.empty((2, n, g), device="cuda")
    assert tb.tb_cuda_group_norm_device(desc, x, gamma, beta, y, mean, rstd, work) == 1
    dy = _normal(gen, n, p, c).to(dtype)
    dx, dgamma, dbeta = torch.empty_like(x), *torch.empty((2, c), device="cuda")
    assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta, work) == 1
    over_x, over_dy, out = x.clone(), dy.clone(), x.clone()
    sums = torch.empty((2, 2, c), device="cuda")
    assert tb.tb_cuda_group_norm_backward_device(desc, over_x, gamma, beta, mean, rstd, dy, over_x, *sums[0], work) == 1
    assert tb.tb_cuda_group_norm_backward_device(desc, x, gamma, beta, mean, rstd, over_dy, over_dy, *sums[1], work) == 1
    assert tb.tb_cuda_group_norm_device(desc, out, gamma, beta, out, None, None, work) == 1
    torch.cuda.synchronize()
    assert torch.equal(over_x, dx) and torch.equal(over_dy, dx) and torch.equal(out, y)
    assert all(torch.equal(s[0], dgamma) and torch.equal(s[1], dbeta) for s in sums)
