"""The learner layers' definitions in 64 bits (torch on any device), written from the formulas of
include/turbinator/training/cuda_learner.h, with bounds on what 32-bit arithmetic may be off.

Each bound is a first-order rounding analysis: U is the unit roundoff of f32, every product, sum or function value
carries a few U of its own magnitude, and magnitudes are the same formulas on absolute values.  A result stored in
fewer bits adds its type's own rounding (`stored`)."""
from __future__ import annotations

import torch

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a unit in the last of 24, 8, 11 bits
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
CHECKPOINT = 16


def stored(ref, error, dtype):
    """Bound on a stored result: the arithmetic's error, then one rounding to `dtype`."""
    return error + ROUND[dtype] * (ref.abs() + error) + LEAST[dtype]


def check(name, got, ref, error):
    """|got - ref| <= the stored bound everywhere; NaN and infinities where the reference has them."""
    got64 = got.double().to(ref.device)
    assert torch.equal(torch.isnan(got64), torch.isnan(ref)), f"{name}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(got64[inf], ref[inf]), f"{name}: infinities differ"
    fine = torch.isfinite(ref)
    off = (got64 - ref).abs()[fine] - stored(ref, error, got.dtype)[fine]
    assert not off.numel() or off.max() <= 0, f"{name}: {int((off > 0).sum())} of {off.numel()} past the bound, by {off.max():.3g}"


# ---- group norm ----

def activate(u, act):
    if act == "silu":
        return u * torch.sigmoid(u)
    if act == "gelu":
        return 0.5 * u * (1 + torch.erf(u / 2 ** 0.5))
    return torch.relu(u) if act == "relu" else u


def group_norm(x, gamma, beta, groups, epsilon, act):
    """x [samples, positions, channels] in 64 bits; y, mean, rstd."""
    n, p, c = x.shape
    byg = x.reshape(n, p, groups, c // groups)
    mean = byg.mean((1, 3))
    rstd = 1 / torch.sqrt(((byg - mean[:, None, :, None]) ** 2).mean((1, 3)) + epsilon)
    hat = ((byg - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(n, p, c)
    return activate(hat * gamma + beta, act), mean, rstd


def _wide(v, per):
    return v.repeat_interleave(per, 1)[:, None]


def group_norm_errors(x, gamma, beta, groups, epsilon, act):
    """Bounds for y, mean, rstd.  A sum of n values in partial sums of at most 64 terms has a relative error below
    (64 + log2 n) U; 128 U covers it with the mean's division."""
    n, p, c = x.shape
    per = c // groups
    _, mean, rstd = group_norm(x, gamma, beta, groups, epsilon, act)
    size = x.abs().reshape(n, p, groups, per).mean((1, 3))
    mean_e = 128 * U * size
    # variance: 2 (x-mean) dmean averages out to dmean^2; each square is 3 U off, each difference U (|x|+|mean|)
    var = 1 / rstd ** 2
    var_e = 160 * U * var + 4 * U * size / rstd + mean_e ** 2
    rstd_e = 0.5 * rstd ** 3 * var_e + 4 * U * rstd
    hat = (x - _wide(mean, per)) * _wide(rstd, per)
    hat_e = _wide(rstd * mean_e, per) + _wide(rstd_e / rstd, per) * hat.abs() + 4 * U * (hat.abs() + _wide(rstd * mean.abs(), per))
    u = hat * gamma + beta
    u_e = gamma.abs() * hat_e + 4 * U * (gamma * hat).abs() + 2 * U * beta.abs()
    # every activation has a slope below 1.2; its own arithmetic is within 16 U of |u| (exp of |u|: |u| U more)
    return 1.2 * u_e + (16 + u.abs().clamp(max=100)) * U * u.abs(), mean_e, rstd_e


def group_norm_backward(x, gamma, beta, mean, rstd, dy, groups, act):
    """dx, dgamma, dbeta and bounds for them, from the given statistics."""
    n, p, c = x.shape
    per = c // groups
    hat = (x - _wide(mean, per)) * _wide(rstd, per)
    u = (hat * gamma + beta).detach().requires_grad_(True)
    du = torch.autograd.grad(activate(u, act), u, dy)[0]
    u = u.detach()
    group = lambda v: _wide(v.reshape(n, p, groups, per).mean((1, 3)), per)  # noqa: E731
    dhat = du * gamma
    dx = _wide(rstd, per) * (dhat - group(dhat) - hat * group(dhat * hat))
    hat_e = 4 * U * (hat.abs() + _wide(rstd * (mean.abs()), per) + _wide(rstd, per) * x.abs())
    u_e = gamma.abs() * hat_e + 4 * U * (gamma * hat).abs() + 2 * U * beta.abs()
    # the slopes change by at most 1 per unit of u (silu 0.5, gelu 0.8); relu's jump is left to inputs away from 0
    du_e = dy.abs() * (u_e * (act != "relu") + (16 + u.abs().clamp(max=100)) * U * 1.2)
    dhat_e = du_e * gamma.abs() + 2 * U * dhat.abs()
    sum_e = lambda v, e: group(e) + 160 * U * group(v.abs())  # noqa: E731
    s2 = group(dhat * hat)
    s2_e = sum_e(dhat * hat, dhat_e * hat.abs() + dhat.abs() * hat_e)
    dx_e = _wide(rstd, per) * (dhat_e + sum_e(dhat, dhat_e) + hat.abs() * s2_e + hat_e * s2.abs() +
                               8 * U * (dhat.abs() + group(dhat).abs() + (hat * s2).abs()))
    total = lambda v: v.sum((0, 1))  # noqa: E731
    dgamma_e = total(du_e * hat.abs() + du.abs() * hat_e) + 256 * U * total((du * hat).abs())
    return (dx, total(du * hat), total(du)), (dx_e, dgamma_e, total(du_e) + 256 * U * total(du.abs()))


# ---- gated recurrence ----

def recurrence(x, rec, inp, decay, scale, reset, lengths, state, dh=None, dstate=None):
    """The recurrence step by step in 64 bits, and with dh its gradients.  Returns {name: (value, bound)}."""
    b, t, d = x.shape
    dev = x.device
    live = torch.arange(t, device=dev)[None] < (lengths[:, None] if lengths is not None else t)
    live = live.expand(b, t)[..., None]
    anew = (reset != 0)[..., None] if reset is not None else torch.zeros((b, t, 1), dtype=torch.bool, device=dev)
    x, rec, inp = (torch.where(live, v, torch.zeros_like(v)) for v in (x, rec, inp))
    soft = torch.logaddexp(decay, torch.zeros_like(decay))
    open_, gate = torch.sigmoid(rec), torch.sigmoid(inp)
    log_a = -scale * soft * open_
    a = torch.where(anew, torch.zeros_like(log_a), torch.exp(log_a))
    beta = torch.where(anew, torch.ones_like(log_a), torch.sqrt(-torch.expm1(2 * log_a)))
    u = gate * x
    h, big, err = state, state.abs(), torch.zeros_like(state)
    before, before_big, before_e, out, out_e = [], [], [], [], []
    # gates within 8 U; a's exponent adds 8 |log a| U, beta = sqrt(-expm1) 16 U, the product 4 U more
    for i in range(t):
        before.append(h), before_big.append(big), before_e.append(err)
        on = live[:, i]
        fresh = a[:, i] * big * (6 + 8 * log_a[:, i].abs() * ~anew[:, i]) + 32 * (beta[:, i] * u[:, i]).abs()
        err = torch.where(on, a[:, i] * err + U * fresh, err)
        big = torch.where(on, a[:, i] * big + (beta[:, i] * u[:, i]).abs(), big)
        h = torch.where(on, a[:, i] * h + beta[:, i] * u[:, i], h)
        out.append(torch.where(on, h, torch.zeros_like(h))), out_e.append(torch.where(on, err, torch.zeros_like(err)))
    stack = lambda v: torch.stack(v, 1)  # noqa: E731
    got = {"h": (stack(out), stack(out_e)), "state": (h, err),
           "checkpoints": (stack(before[::CHECKPOINT]), stack(before_e[::CHECKPOINT]))}
    if dh is None:
        return got
    g, big, err = dstate, dstate.abs(), torch.zeros_like(dstate)
    rows = {n: [None] * t for n in ("dx", "drec", "dinp")}
    errs = {n: [None] * t for n in rows}
    dsoft, dsoft_e = torch.zeros_like(decay), torch.zeros_like(decay)
    for i in reversed(range(t)):
        on, keep = live[:, i], ~anew[:, i]
        grad = torch.where(on, dh[:, i], torch.zeros_like(g))
        total, total_big, total_e = g + grad, big + grad.abs(), err + 2 * U * (big + grad.abs())
        ai, bi, ui, xi, ga, op, la = a[:, i], beta[:, i], u[:, i], x[:, i], gate[:, i], open_[:, i], log_a[:, i]
        ratio = torch.where(bi > 0, ai / bi, torch.zeros_like(ai)) * (bi > 0)
        inner, inner_big = before[i] - ratio * ui, before_big[i] + (ratio * ui).abs()
        inner_e = before_e[i] + 40 * U * inner_big
        dlog = ai * total * inner * keep * (bi > 0)
        dlog_e = ai * (total_e * inner_big + total_big * inner_e + (16 + 8 * la.abs()) * U * total_big * inner_big)
        dlog_e = dlog_e * keep * (bi > 0)
        zero = torch.zeros_like(g)
        put = lambda n, v, e: (rows[n].__setitem__(i, torch.where(on, v, zero)),  # noqa: E731
                               errs[n].__setitem__(i, torch.where(on, e, zero)))
        put("dx", total * bi * ga, bi * ga * (total_e + 40 * U * total_big))
        put("dinp", total * bi * ui * (1 - ga), (bi * ui).abs() * (total_e * (1 - ga) + 48 * U * total_big))
        put("drec", dlog * la * (1 - op), la.abs() * (dlog_e * (1 - op) + 24 * U * dlog.abs()))
        dsoft = dsoft + torch.where(on, dlog * op, zero).sum(0)
        dsoft_e = dsoft_e + torch.where(on, op * (dlog_e + 256 * U * dlog.abs()), zero).sum(0)
        g = torch.where(on, ai * total, g)
        err = torch.where(on, ai * total_e + ai * total_big * (4 + 8 * la.abs() * keep) * U, err)
        big = torch.where(on, ai * total_big, big)
    slope = scale * torch.sigmoid(decay)
    for n in rows:
        got[n] = (stack(rows[n]), stack(errs[n]))
    got["ddecay"] = (-slope * dsoft, slope * (dsoft_e + 16 * U * dsoft.abs()))
    got["dstate"] = (g, err)
    return got


# ---- routing ----

def available(logits):
    return torch.where(torch.isnan(logits), torch.full_like(logits, float("-inf")), logits)


def scores(logits, kind):
    """Scores of [tokens, experts] logits: softmax over the available experts (a +inf logit shares with its like)."""
    if kind == "sigmoid":
        return torch.where(logits > float("-inf"), torch.sigmoid(logits), torch.zeros_like(logits))
    top = logits.amax(1, keepdim=True).detach()
    e = torch.exp(torch.where(torch.isinf(top) & (logits == top), torch.zeros_like(logits), logits - top))
    e = torch.where(logits > float("-inf"), e, torch.zeros_like(e))
    return e / e.sum(1, keepdim=True).clamp(min=1e-300)


def route(logits, bias, kind, top_k, groups=1, top_groups=1, group_best=1, renormalise=False, scale=1.0):
    """ids, weights (64 bits), and each token's smallest gap between two ranking values that a comparison uses."""
    logits = available(logits.double())
    t, e = logits.shape
    score = scores(logits, kind)
    neg = float("-inf")
    ids = torch.full((t, top_k), -1, dtype=torch.int64)
    gap = torch.full((t,), float("inf"), dtype=torch.float64)
    for r in range(t):
        free = [i for i in range(e) if logits[r, i] > neg]
        rank = {i: float(score[r, i]) + float(bias[i]) if bias is not None else float(logits[r, i]) for i in free}
        plain = bias is None and not (groups > 1 and group_best == 2)
        by_group = rank if plain or bias is not None else {i: float(score[r, i]) for i in free}
        if groups > 1:
            per = e // groups
            strength = []
            for g in range(groups):
                vals = sorted((by_group[i] for i in free if i // per == g), reverse=True)
                strength.append(sum(vals[:group_best]) if vals else neg)
            order = sorted(range(groups), key=lambda g: (-strength[g], g))
            if top_groups < groups and strength[order[top_groups]] > neg:
                d = strength[order[top_groups - 1]] - strength[order[top_groups]]
                gap[r] = min(float(gap[r]), d if d > 0 else float("inf") if plain else d)
            kept = set(order[:top_groups])
            free = [i for i in free if i // per in kept]
        order = sorted(free, key=lambda i: (-rank[i], i))
        for a, b in zip(order[:top_k], order[1:top_k + 1]):
            if bias is not None:
                gap[r] = min(float(gap[r]), rank[a] - rank[b])
        ids[r, :min(top_k, len(order))] = torch.tensor(order[:top_k], dtype=torch.int64)
    picked = torch.where(ids >= 0, score.gather(1, ids.clamp(min=0)), 0.0)
    if renormalise:
        total = picked.sum(1, keepdim=True)
        picked = torch.where(total > 0, picked / total, 0.0)
    return ids, picked * scale, gap


def slot_lists(ids, experts):
    """offsets, order, position of the slots with an expert."""
    flat = ids.reshape(-1).tolist()
    order = sorted((i for i, e in enumerate(flat) if e >= 0), key=lambda i: (flat[i], i))
    offsets = [sum(1 for e in flat if 0 <= e < k) for k in range(experts + 1)]
    position = [-1] * len(flat)
    for place, i in enumerate(order):
        position[i] = place
    return offsets, order + [-1] * (len(flat) - len(order)), position


def route_weights(logits, ids, kind, renormalise, scale):
    """The weights of given ids, differentiable in the logits (the selection is fixed)."""
    score = scores(logits, kind)
    picked = torch.where(ids >= 0, score.gather(1, ids.clamp(min=0)), 0.0)
    if renormalise:
        total = picked.sum(1, keepdim=True)
        picked = torch.where(total > 0, picked / total.clamp(min=1e-300), 0.0)
    return picked * scale
