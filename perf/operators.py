"""The learner operators as workloads: group norm with an activation, the gated recurrence, expert routing and the
expert combine, each in a plain form of elementary torch operations and through this package's entry points.

The library hands a learner its input tensors (proprio, LiDAR channels, camera luma).  The layers that read them are
convolution stems with group norm, a recurrence over each aircraft's trajectory, and a trunk of routed experts; the
cases below are those layers at acting size (a few aircraft, one step) and at training size (whole trajectories)."""
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
CHECKPOINT = 16  # steps between two saved states of the recurrence
DECAY_SCALE = 8.0
EPSILON = 1e-5


def listed():
    return [
        # acting: the camera stem of 8 aircraft (4 views each), one 16x16 map of 32 channels per view
        dict(name="norm_act_8_aircraft", op="norm", back=False, samples=32, positions=256, channels=32, groups=8,
             act="silu", type="f32", pad=0),
        # few and large maps: 8 images of 256x256, far more than a cluster's shared memory per image
        dict(name="norm_large_maps", op="norm", back=False, samples=8, positions=65536, channels=128, groups=32,
             act="silu", type="bf16", pad=0),
        # training: the backward pass of the stem over 1,024 aircraft x 4 views
        dict(name="norm_train_backward", op="norm", back=True, samples=4096, positions=256, channels=64, groups=8,
             act="silu", type="bf16", pad=0),
        # acting: one step of 64 aircraft from their kept states
        dict(name="recurrence_step", op="recurrence", back=False, sequences=64, steps=1, channels=512, type="bf16",
             resets=False, ragged=False, train=False),
        # training: 64 trajectories of 1,024 steps with episode ends inside them
        dict(name="recurrence_train", op="recurrence", back=False, sequences=64, steps=1024, channels=1024,
             type="bf16", resets=True, ragged=False, train=True),
        dict(name="recurrence_train_backward", op="recurrence", back=True, sequences=64, steps=1024, channels=1024,
             type="bf16", resets=True, ragged=False, train=True),
        # three long logs of unequal lengths through a narrow odd layer: few channels, many steps
        dict(name="recurrence_long_logs", op="recurrence", back=False, sequences=3, steps=30011, channels=321,
             type="f32", resets=False, ragged=True, train=False),
        # acting: 61 aircraft, sigmoid scores with a balance bias, experts in groups
        dict(name="route_act", op="route", back=False, tokens=61, experts=64, top_k=6, groups=8, top_groups=3,
             score="sigmoid", bias=True, renormalise=True, masked=0.0, type="f32"),
        # training: every step of the trajectories above, a quarter of them padding, softmax scores
        dict(name="route_train", op="route", back=False, tokens=65536, experts=256, top_k=8, groups=1, top_groups=1,
             score="softmax", bias=False, renormalise=True, masked=0.25, type="bf16"),
        dict(name="route_train_backward", op="route", back=True, tokens=65536, experts=256, top_k=8, groups=1,
             top_groups=1, score="sigmoid", bias=True, renormalise=True, masked=0.0, type="bf16"),
        # the experts' outputs back to their tokens, and its gradient
        dict(name="combine_small", op="combine", back=False, tokens=61, top_k=6, width=520, type="f32"),
        dict(name="combine_train_backward", op="combine", back=True, tokens=16384, top_k=8, width=1024, type="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "recurrence", "route", "combine"])
    kind = rng.choice(["f32", "bf16", "bf16", "f16"])
    back = rng.random() < 0.5
    if op == "norm":
        groups = rng.choice([1, 2, 4, 8, 8, 16, 32, 12])
        channels = groups * rng.choice([1, 2, 3, 4, 4, 7, 8, 8, 16])
        positions = _spread(rng, 8, 65536)
        samples = _spread(rng, 1, max(1, min(8192, 40_000_000 // (positions * channels))))
        return dict(op=op, back=back, samples=samples, positions=positions, channels=channels, groups=groups,
                    act=rng.choice(["none", "relu", "silu", "silu", "gelu"]), type=kind, pad=rng.choice([0, 0, 8, 3]))
    if op == "recurrence":
        channels = rng.choice([_spread(rng, 4, 2048), 64 * _spread(rng, 1, 32)])
        steps = _spread(rng, 1, 65536)
        sequences = _spread(rng, 1, max(1, min(4096, 30_000_000 // (steps * channels))))
        return dict(op=op, back=back, sequences=sequences, steps=steps, channels=channels, type=kind,
                    resets=rng.random() < 0.5, ragged=rng.random() < 0.5, train=back or rng.random() < 0.5)
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _spread(rng, 2, 512 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, top_groups * (experts // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        return dict(op=op, back=back, tokens=_spread(rng, 1, 65536 if experts <= 256 else 32768), experts=experts,
                    top_k=top_k, groups=groups, top_groups=top_groups, score=score,
                    bias=score == "sigmoid" and rng.random() < 0.7, renormalise=top_k > 1 and rng.random() < 0.7,
                    masked=rng.choice([0.0, 0.3]), type=kind)
    top_k = rng.randint(1, 12)
    width = rng.choice([_spread(rng, 1, 2048), 128 * rng.randint(1, 16)])
    return dict(op=op, back=back, tokens=_spread(rng, 1, max(1, min(65536, 60_000_000 // (top_k * width)))),
                top_k=top_k, width=width, type=kind)


# ---- inputs ----

def _normal(shape, gen, scale=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda") * scale + mean


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"norm": _prepare_norm, "recurrence": _prepare_recurrence, "route": _prepare_route,
             "combine": _prepare_combine}[case["op"]](case, gen)
    state["case"] = case
    if own:  # what a user's program keeps between calls: the descriptor, the workspace and the output buffers
        _plan(case, state)
    return state


def _prepare_norm(case, gen):
    n, p, c, g = (case[k] for k in ("samples", "positions", "channels", "groups"))
    kind = TYPES[case["type"]]
    # `pad` > 0: the normalised channels are a slice of a wider map
    x = _normal((n, p, c + case["pad"]), gen, 1.3, 0.4).to(kind)[..., :c]
    s = {"x": x, "gamma": _normal((c,), gen, 0.2, 1.0), "beta": _normal((c,), gen, 0.2)}
    if case["back"]:
        x32 = x.float().reshape(n, p, g, c // g)
        mean = x32.mean((1, 3))
        s["mean"] = mean
        s["rstd"] = ((x32 - mean[:, None, :, None]).square().mean((1, 3)) + EPSILON).rsqrt()
        s["dy"] = _normal((n, p, c), gen).to(kind)
    return s


def _prepare_recurrence(case, gen):
    b, t, d = (case[k] for k in ("sequences", "steps", "channels"))
    kind = TYPES[case["type"]]
    # x and both gates are thirds of one projection's output
    xgg = _normal((b, t, 3 * d), gen).to(kind)
    s = {"x": xgg[..., :d], "rec": xgg[..., d:2 * d], "inp": xgg[..., 2 * d:]}
    keep = torch.rand((d,), generator=gen, device="cuda") * 0.099 + 0.9  # the decay of a fully open gate
    s["decay"] = torch.log(torch.expm1(-torch.log(keep) / DECAY_SCALE))
    s["state"] = _normal((b, d), gen, 0.5)
    s["reset"] = s["lengths"] = None
    if case["resets"]:
        s["reset"] = (torch.rand((b, t), generator=gen, device="cuda") < 1 / 200).to(torch.uint8)
    if case["ragged"]:
        s["lengths"] = torch.randint(t // 2, t + 1, (b,), generator=gen, device="cuda").to(torch.int32)
    if case["back"]:
        log_a, u, scale = _gates(s, t)
        h, _ = _scan(log_a.exp(), u * scale, s["state"])
        before = torch.cat([s["state"][:, None], h[:, :-1]], 1)
        s["checkpoints"] = before[:, ::CHECKPOINT].contiguous()
        s["dh"] = _normal((b, t, d), gen).to(kind)
        s["dstate"] = _normal((b, d), gen)
    return s


def _prepare_route(case, gen):
    t, e, k = (case[n] for n in ("tokens", "experts", "top_k"))
    logits = _normal((t, e), gen, 1.5)
    if case["masked"]:  # padding tokens take no expert: their whole row is minus infinity
        logits[torch.rand((t,), generator=gen, device="cuda") < case["masked"]] = float("-inf")
    s = {"logits": logits.to(TYPES[case["type"]]), "bias": None}
    if case["bias"]:  # the balance bias moves in steps of 0.001
        s["bias"] = torch.randint(-40, 41, (e,), generator=gen, device="cuda") * 0.001
    if case["back"]:
        s["ids"] = _select(case, s["logits"].float(), s["bias"])[0].to(torch.int32)
        s["dweights"] = _normal((t, k), gen)
    return s


def _prepare_combine(case, gen):
    t, k, w = (case[n] for n in ("tokens", "top_k", "width"))
    kind = TYPES[case["type"]]
    s = {"rows": _normal((t * k, w), gen).to(kind), "weights": torch.rand((t, k), generator=gen, device="cuda")}
    s["position"] = torch.randperm(t * k, generator=gen, device="cuda").reshape(t, k).to(torch.int32)
    if case["back"]:
        s["dout"] = _normal((t, w), gen).to(kind)
    return s


# ---- the work that no form can do without ----

def work(case):
    s = SIZE[case["type"]]
    if case["op"] == "norm":
        n = case["samples"] * case["positions"] * case["channels"]
        return {"bytes": n * s * (3 if case["back"] else 2) + 8 * case["samples"] * case["groups"] +
                8 * case["channels"], "flops": n * (30 if case["back"] else 14)}
    if case["op"] == "recurrence":
        n = case["sequences"] * case["steps"] * case["channels"]
        ends = 8 * case["sequences"] * case["channels"] + 4 * case["channels"]
        saved = 4 * n / CHECKPOINT if case["train"] else 0
        flags = case["sequences"] * case["steps"] * case["resets"]
        return {"bytes": n * s * (7 if case["back"] else 4) + saved + ends + flags,
                "flops": n * (45 if case["back"] else 20)}
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        if case["back"]:
            return {"bytes": 2 * t * e * s + 8 * t * k, "flops": 8 * t * e}
        return {"bytes": t * e * s + 16 * t * k + 4 * e, "flops": 6 * t * e}
    n = case["tokens"] * case["width"]
    slots = case["tokens"] * case["top_k"]
    if case["back"]:
        return {"bytes": n * s + 2 * n * case["top_k"] * s + 12 * slots, "flops": 3 * n * case["top_k"]}
    return {"bytes": n * s + n * case["top_k"] * s + 8 * slots, "flops": 2 * n * case["top_k"]}


# ---- one pass ----

def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"], case["back"]](state)
    return _PLAIN[case["op"], case["back"]](case, state)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end ----

def _act(u, name):
    if name == "silu":
        return u / (1 + torch.exp(-u))
    if name == "gelu":
        return 0.5 * u * (1 + torch.erf(u * 0.5 ** 0.5))
    return u.clamp(min=0) if name == "relu" else u


def _act_slope(u, name):
    if name == "silu":
        sig = 1 / (1 + torch.exp(-u))
        return sig * (1 + u * (1 - sig))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(u * 0.5 ** 0.5)) + u * torch.exp(-0.5 * u * u) * 0.3989422804014327
    return (u > 0).to(u.dtype) if name == "relu" else torch.ones_like(u)


def _plain_norm(case, s):
    n, p, c, g = (case[k] for k in ("samples", "positions", "channels", "groups"))
    x = s["x"].float().reshape(n, p, g, c // g)
    mean = x.mean((1, 3))
    off = x - mean[:, None, :, None]
    rstd = 1 / torch.sqrt((off * off).mean((1, 3)) + EPSILON)
    u = (off * rstd[:, None, :, None]).reshape(n, p, c) * s["gamma"] + s["beta"]
    return {"y": _act(u, case["act"]).to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_norm_back(case, s):
    n, p, c, g = (case[k] for k in ("samples", "positions", "channels", "groups"))
    rstd = s["rstd"][:, None, :, None]
    hat = (s["x"].float().reshape(n, p, g, c // g) - s["mean"][:, None, :, None]) * rstd
    flat = hat.reshape(n, p, c)
    du = s["dy"].float() * _act_slope(flat * s["gamma"] + s["beta"], case["act"])
    dhat = (du * s["gamma"]).reshape(n, p, g, c // g)
    dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    return {"dx": dx.reshape(n, p, c).to(s["x"].dtype), "dgamma": (du * flat).sum((0, 1)), "dbeta": du.sum((0, 1))}


def _gates(s, steps):
    """log a [B,T,D], the gated input and its scale sqrt(1 - a^2); a step that is a reset forgets all before it, and a
    step past its sequence's length changes nothing."""
    open_ = 1 / (1 + torch.exp(-s["rec"].float()))
    log_a = -DECAY_SCALE * torch.log1p(torch.exp(s["decay"])) * open_
    u = s["x"].float() / (1 + torch.exp(-s["inp"].float()))
    if s["reset"] is not None:
        log_a = log_a.masked_fill(s["reset"][..., None] != 0, float("-inf"))
    scale = torch.sqrt(-torch.expm1(2 * log_a))
    if s["lengths"] is not None:
        past = (torch.arange(steps, device="cuda") >= s["lengths"][:, None])[..., None]
        log_a, u = log_a.masked_fill(past, 0.0), u.masked_fill(past, 0.0)
        scale = scale.masked_fill(past, 0.0)
    return log_a, u, scale


def _scan(a, b, first):
    """h_t = a_t h_(t-1) + b_t along dim 1, by doubling; returns h and a buffer that it used."""
    b = b.clone()
    b[:, 0] += a[:, 0] * first
    span, steps = 1, b.shape[1]
    while span < steps:  # after each turn a and b cover spans of twice the length
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b, a


def _plain_recurrence(case, s):
    kind, steps = s["x"].dtype, case["steps"]
    log_a, u, scale = _gates(s, steps)
    h, _ = _scan(log_a.exp(), u * scale, s["state"])
    out = {"state": h[:, -1].clone()}
    if case["train"]:
        out["checkpoints"] = torch.cat([s["state"][:, None], h[:, CHECKPOINT - 1:-1:CHECKPOINT]], 1)
    if s["lengths"] is not None:
        past = (torch.arange(steps, device="cuda") >= s["lengths"][:, None])[..., None]
        h = h.masked_fill(past, 0.0)
    out["h"] = h.to(kind)
    return out


def _plain_recurrence_back(case, s):
    kind, steps = s["x"].dtype, case["steps"]
    log_a, u, scale = _gates(s, steps)
    a = log_a.exp()
    h, _ = _scan(a, u * scale, s["state"])
    before = torch.cat([s["state"][:, None], h[:, :-1]], 1)
    dh = s["dh"].float()
    if s["lengths"] is not None:
        past = (torch.arange(steps, device="cuda") >= s["lengths"][:, None])[..., None]
        dh = dh.masked_fill(past, 0.0)
    # backwards in time: c_t = a_t (dh_t + c_(t+1)), the gradient of the state before step t
    c, _ = _scan(a.flip(1), (a * dh).flip(1), s["dstate"])
    c = c.flip(1)
    g = dh + torch.cat([c[:, 1:], s["dstate"][:, None]], 1)
    open_ = 1 / (1 + torch.exp(-s["rec"].float()))
    gate = 1 / (1 + torch.exp(-s["inp"].float()))
    dlog_a = g * a * (before - torch.where(scale > 0, a / scale, 0 * scale) * u)
    drec = torch.where(a > 0, dlog_a * log_a * (1 - open_), 0 * a)
    soft = torch.log1p(torch.exp(s["decay"]))
    dsoft = torch.where((a > 0) & (log_a < 0), dlog_a * open_, 0 * a).sum((0, 1)) * -DECAY_SCALE
    dx = g * scale * gate
    if s["lengths"] is not None:
        dx = dx.masked_fill(past, 0.0)
    return {"dx": dx.to(kind), "drec": drec.to(kind), "dinp": (g * scale * u * (1 - gate)).to(kind),
            "ddecay": dsoft * -torch.expm1(-soft), "dstate": c[:, 0].clone()}


def _select(case, logits, bias):
    """The experts of each token, best first (ties: the lower index), and their scores; -1 and 0 where none is left.
    Without a bias a score's order is its logit's."""
    t, e = logits.shape
    groups, k = case["groups"], case["top_k"]
    free = logits > float("-inf")
    if case["score"] == "softmax":
        score = torch.exp(logits - logits.amax(1, keepdim=True).clamp(min=-3e38))
        score = score / score.sum(1, keepdim=True).clamp(min=1e-38)
        value = logits
    else:
        score = 1 / (1 + torch.exp(-logits))
        value = score + bias if bias is not None else score if groups > 1 else logits
    value = value.masked_fill(~free, float("-inf"))
    if groups > 1:
        parts = value.reshape(t, groups, e // groups)
        if case["score"] == "softmax":  # a group's best expert
            strength = parts.amax(2)
        else:  # the sum of a group's two best (one that is not there adds nothing)
            best = parts.sort(dim=2, descending=True)[0]
            second = best[..., 1] if e > groups else torch.full_like(best[..., 0], float("-inf"))
            strength = best[..., 0] + torch.where(second > float("-inf"), second, 0.0)
        chosen = strength.sort(dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        inside = torch.zeros_like(strength, dtype=torch.bool).scatter_(1, chosen, True)
        inside = inside & (strength > float("-inf"))
        free = free & inside.repeat_interleave(e // groups, 1)
        if case["score"] == "sigmoid" and bias is None:
            value = logits
        value = value.masked_fill(~free, float("-inf"))
    ids = value.sort(dim=1, descending=True, stable=True)[1][:, :k]
    taken = free.gather(1, ids)
    return torch.where(taken, ids, -1), torch.where(taken, score.gather(1, ids), 0.0), score


def _plain_route(case, s):
    t, e, k = (case[n] for n in ("tokens", "experts", "top_k"))
    ids, picked, _ = _select(case, s["logits"].float(), s["bias"])
    total = picked.sum(1, keepdim=True)
    weights = torch.where(total > 0, picked / total, 0.0) if case["renormalise"] else picked
    flat = ids.reshape(-1)
    key = torch.where(flat >= 0, flat, e)
    key, order = key.sort(dim=0, stable=True)
    offsets = torch.searchsorted(key, torch.arange(e + 1, device="cuda"))
    taken = key < e
    place = torch.where(taken, torch.arange(t * k, device="cuda"), -1)
    position = torch.empty_like(place)
    position[order] = place
    return {"ids": ids.to(torch.int32), "weights": weights, "offsets": offsets.to(torch.int32),
            "order": torch.where(taken, order, -1).to(torch.int32),
            "position": position.reshape(t, k).to(torch.int32)}


def _plain_route_back(case, s):
    logits, ids = s["logits"].float(), s["ids"].long()
    taken = ids >= 0
    at = ids.clamp(min=0)
    if case["score"] == "softmax":
        score = torch.exp(logits - logits.amax(1, keepdim=True).clamp(min=-3e38))
        score = score / score.sum(1, keepdim=True).clamp(min=1e-38)
    else:
        score = 1 / (1 + torch.exp(-logits))
    picked = torch.where(taken, score.gather(1, at), 0.0)
    dpicked = torch.where(taken, s["dweights"], 0.0)
    if case["renormalise"]:
        total = picked.sum(1, keepdim=True)
        inner = torch.where(total > 0, (dpicked * picked).sum(1, keepdim=True) / total, 0.0)
        dpicked = torch.where(taken & (total > 0), (dpicked - inner) / total, 0.0)
    dscore = torch.zeros_like(score).scatter_add_(1, at, dpicked)
    if case["score"] == "softmax":
        dlogits = score * (dscore - (dscore * score).sum(1, keepdim=True))
    else:
        dlogits = dscore * score * (1 - score)
    return {"dlogits": dlogits.to(s["logits"].dtype)}


def _plain_combine(case, s):
    rows = s["rows"].float()[s["position"].long()]
    return {"out": (rows * s["weights"][..., None]).sum(1).to(s["rows"].dtype)}


def _plain_combine_back(case, s):
    at = s["position"].long()
    dout = s["dout"].float()[:, None]
    drows = torch.empty_like(s["rows"])
    drows[at.reshape(-1)] = (dout * s["weights"][..., None]).reshape(-1, case["width"]).to(drows.dtype)
    return {"drows": drows, "dweights": (dout * s["rows"].float()[at]).sum(2)}


_PLAIN = {("norm", False): _plain_norm, ("norm", True): _plain_norm_back,
          ("recurrence", False): _plain_recurrence, ("recurrence", True): _plain_recurrence_back,
          ("route", False): _plain_route, ("route", True): _plain_route_back,
          ("combine", False): _plain_combine, ("combine", True): _plain_combine_back}


# ---- this package's entry points ----

def _plan(case, s):
    import turbinator_c_b200 as tb

    kind = {"f32": tb.TB_TYPE_F32, "bf16": tb.TB_TYPE_BF16, "f16": tb.TB_TYPE_F16}[case["type"]]
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    s["tb"], need = tb, 0
    if case["op"] == "norm":
        n, p, c, g = (case[k] for k in ("samples", "positions", "channels", "groups"))
        act = {"none": tb.TB_ACT_NONE, "relu": tb.TB_ACT_RELU, "silu": tb.TB_ACT_SILU, "gelu": tb.TB_ACT_GELU}
        # x as it lies; y, dy and dx dense
        s["plan"] = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=kind,
                                     activation=act[case["act"]], epsilon=EPSILON,
                                     x_sample_stride=p * (c + case["pad"]), x_position_stride=c + case["pad"])
        need = tb.tb_cuda_group_norm_workspace(s["plan"])
        if case["back"]:
            s["out"] = {"dx": new(n, p, c, dtype=s["x"].dtype), "dgamma": new(c), "dbeta": new(c)}
        else:
            s["out"] = {"y": new(n, p, c, dtype=s["x"].dtype), "mean": new(n, g), "rstd": new(n, g)}
    elif case["op"] == "recurrence":
        b, t, d = (case[k] for k in ("sequences", "steps", "channels"))
        s["plan"] = tb.GatedRecurrenceDesc(sequences=b, steps=t, channels=d, type=kind, decay_scale=DECAY_SCALE,
                                           in_sequence_stride=t * 3 * d, in_step_stride=3 * d)
        need = tb.tb_cuda_gated_recurrence_workspace(s["plan"])
        like = s["x"].dtype
        if case["back"]:
            s["out"] = {"dx": new(b, t, d, dtype=like), "drec": new(b, t, d, dtype=like),
                        "dinp": new(b, t, d, dtype=like), "ddecay": new(d), "dstate": new(b, d)}
        else:
            s["out"] = {"h": new(b, t, d, dtype=like), "state": new(b, d)}
            if case["train"]:
                s["out"]["checkpoints"] = new(b, -(-t // CHECKPOINT), d)
    elif case["op"] == "route":
        t, e, k = (case[n] for n in ("tokens", "experts", "top_k"))
        soft = case["score"] == "softmax"
        s["plan"] = tb.ExpertRouteDesc(tokens=t, experts=e, top_k=k, groups=case["groups"],
                                       top_groups=case["top_groups"], group_best=1 if soft else 2, type=kind,
                                       score=tb.TB_SCORE_SOFTMAX if soft else tb.TB_SCORE_SIGMOID,
                                       renormalise=int(case["renormalise"]), weight_scale=1.0)
        need = tb.tb_cuda_route_experts_workspace(s["plan"])
        whole = torch.int32
        if case["back"]:
            s["out"] = {"dlogits": new(t, e, dtype=s["logits"].dtype)}
        else:
            s["out"] = {"ids": new(t, k, dtype=whole), "weights": new(t, k), "offsets": new(e + 1, dtype=whole),
                        "order": new(t * k, dtype=whole), "position": new(t, k, dtype=whole)}
    else:
        t, k, w = (case[n] for n in ("tokens", "top_k", "width"))
        s["plan"] = tb.ExpertCombineDesc(tokens=t, top_k=k, rows=t * k, width=w, type=kind)
        if case["back"]:
            s["out"] = {"drows": new(t * k, w, dtype=s["rows"].dtype), "dweights": new(t, k)}
        else:
            s["out"] = {"out": new(t, w, dtype=s["rows"].dtype)}
    s["workspace"] = new(max(1, need), dtype=torch.uint8)


def _checked(ok):
    if ok != 1:
        raise RuntimeError("the call was refused")


def _own_norm(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_group_norm_device(s["plan"], s["x"], s["gamma"], s["beta"], o["y"], o["mean"], o["rstd"],
                                               s["workspace"], torch.cuda.current_stream()))
    return o


def _own_norm_back(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_group_norm_backward_device(
        s["plan"], s["x"], s["gamma"], s["beta"], s["mean"], s["rstd"], s["dy"], o["dx"], o["dgamma"], o["dbeta"],
        s["workspace"], torch.cuda.current_stream()))
    return o


def _own_recurrence(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_gated_recurrence_device(
        s["plan"], s["x"], s["rec"], s["inp"], s["decay"], s["reset"], s["lengths"], s["state"], o["h"], o["state"],
        o.get("checkpoints"), s["workspace"], torch.cuda.current_stream()))
    return o


def _own_recurrence_back(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_gated_recurrence_backward_device(
        s["plan"], s["x"], s["rec"], s["inp"], s["decay"], s["reset"], s["lengths"], s["checkpoints"], s["dh"],
        s["dstate"], o["dx"], o["drec"], o["dinp"], o["ddecay"], o["dstate"], s["workspace"],
        torch.cuda.current_stream()))
    return o


def _own_route(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_route_experts_device(s["plan"], s["logits"], s["bias"], o["ids"], o["weights"],
                                                  o["offsets"], o["order"], o["position"], s["workspace"],
                                                  torch.cuda.current_stream()))
    return o


def _own_route_back(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_route_experts_backward_device(s["plan"], s["logits"], s["ids"], s["dweights"],
                                                           o["dlogits"], torch.cuda.current_stream()))
    return o


def _own_combine(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_combine_experts_device(s["plan"], s["rows"], s["position"], s["weights"], o["out"],
                                                    torch.cuda.current_stream()))
    return o


def _own_combine_back(s):
    o = s["out"]
    _checked(s["tb"].tb_cuda_combine_experts_backward_device(
        s["plan"], s["rows"], s["position"], s["weights"], s["dout"], o["drows"], o["dweights"],
        torch.cuda.current_stream()))
    return o


_OWN = {("norm", False): _own_norm, ("norm", True): _own_norm_back,
        ("recurrence", False): _own_recurrence, ("recurrence", True): _own_recurrence_back,
        ("route", False): _own_route, ("route", True): _own_route_back,
        ("combine", False): _own_combine, ("combine", True): _own_combine_back}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "recurrence": _exact_recurrence, "route": _exact_route,
            "combine": _exact_combine}[case["op"]](case, s)


def _exact_norm(case, s):
    n, p, c, g = (case[k] for k in ("samples", "positions", "channels", "groups"))
    per = c // g
    got = {"y": [], "dx": []}
    means, rstds = [], []
    gamma, beta = s["gamma"].double(), s["beta"].double()
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    step = max(1, 100_000_000 // (p * c))
    for i in range(0, n, step):
        x = s["x"][i:i + step].double()
        byg = x.unflatten(2, (g, per)).transpose(1, 2).flatten(2)  # [samples, groups, positions * per]
        if case["back"]:  # the saved statistics are inputs of the backward pass
            mean, rstd = s["mean"][i:i + step].double(), s["rstd"][i:i + step].double()
        else:
            var, mean = torch.var_mean(byg, 2, correction=0)
            rstd = (var + EPSILON).pow(-0.5)
        wide = lambda v: v.repeat_interleave(per, 1)[:, None]  # noqa: E731
        hat = (x - wide(mean)) * wide(rstd)
        u = hat * gamma + beta
        u.requires_grad_(True)
        y = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
             "none": lambda v: v * 1.0}[case["act"]](u)
        if not case["back"]:
            got["y"].append(y.detach())
            means.append(mean)
            rstds.append(rstd)
            continue
        du = torch.autograd.grad(y, u, s["dy"][i:i + step].double())[0]
        dgamma += (du * hat).sum((0, 1))
        dbeta += du.sum((0, 1))
        dhat = du * gamma
        sums = lambda v: wide(v.sum(1).unflatten(1, (g, per)).sum(2) / (p * per))  # noqa: E731
        got["dx"].append(wide(rstd) * (dhat - sums(dhat) - hat * sums(dhat * hat)))
    if case["back"]:
        return {"dx": torch.cat(got["dx"]), "dgamma": dgamma, "dbeta": dbeta}
    return {"y": torch.cat(got["y"]), "mean": torch.cat(means), "rstd": torch.cat(rstds)}


def _exact_recurrence(case, s):
    b, t, d = (case[k] for k in ("sequences", "steps", "channels"))
    live = torch.ones((b, t), dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        live = torch.arange(t, device="cuda") < s["lengths"][:, None]
    kept = torch.ones((b, t), dtype=torch.float64, device="cuda")
    if s["reset"] is not None:
        kept = (s["reset"] == 0).double()
    soft = torch.nn.functional.softplus(s["decay"].double(), threshold=1000)
    h = s["state"].double()
    out, saved, was = [], [], []

    def step(i):
        r = torch.sigmoid(s["rec"][:, i].double())
        a = torch.exp(-DECAY_SCALE * soft * r) * kept[:, i, None]
        return r, a, torch.sigmoid(s["inp"][:, i].double())

    for i in range(t):
        _, a, gate = step(i)
        was.append(h if case["back"] else None)
        if i % CHECKPOINT == 0:
            saved.append(h)
        new = a * h + torch.sqrt((1 - a) * (1 + a)) * gate * s["x"][:, i].double()
        h = torch.where(live[:, i, None], new, h)
        out.append(torch.where(live[:, i, None], new, 0.0).float() if t * b * d > 60_000_000 else
                   torch.where(live[:, i, None], new, 0.0))
    if not case["back"]:
        got = {"h": torch.stack(out, 1), "state": h}
        if case["train"]:
            got["checkpoints"] = torch.stack(saved, 1)
        return got
    del out
    g = s["dstate"].double()  # the gradient of the state after step i
    dsoft = torch.zeros((d,), dtype=torch.float64, device="cuda")
    dx, drec, dinp = [], [], []
    for i in reversed(range(t)):
        r, a, gate = step(i)
        on = live[:, i, None]
        total = torch.where(on, g + s["dh"][:, i].double(), 0.0)
        beta = torch.sqrt((1 - a) * (1 + a))
        x = s["x"][:, i].double()
        dlog = total * a * (was[i] - torch.where(beta > 0, a / beta, 0.0) * gate * x) * kept[:, i, None]
        dx.append((total * beta * gate).float())
        dinp.append((total * beta * x * gate * (1 - gate)).float())
        drec.append((dlog * -DECAY_SCALE * soft * r * (1 - r)).float())
        dsoft += (dlog * r).sum(0) * -DECAY_SCALE
        g = torch.where(on, total * a, g)
        was[i] = None
    # what is rounded to 16 bits in the end is held in 32 here, for memory
    return {"dx": torch.stack(dx[::-1], 1), "drec": torch.stack(drec[::-1], 1), "dinp": torch.stack(dinp[::-1], 1),
            "ddecay": dsoft * torch.sigmoid(s["decay"].double()), "dstate": g}


def _exact_route(case, s):
    logits = s["logits"].double()
    t, e, k = (case[n] for n in ("tokens", "experts", "top_k"))
    score = torch.nan_to_num(logits.softmax(1)) if case["score"] == "softmax" else logits.sigmoid()
    if case["back"]:
        at = s["ids"].long()
    else:
        rank = score + s["bias"].double() if s["bias"] is not None else score
        rank = torch.where(torch.isinf(logits), -1e300, rank)
        if case["groups"] > 1:
            two = rank.unflatten(1, (case["groups"], -1)).topk(1 if case["score"] == "softmax" else 2, 2)[0]
            best = torch.cat([two[..., :1], two[..., 1:].clamp(min=-1e250) * (two[..., 1:] > -1e299)], 2).sum(2)
            worse = best.argsort(dim=1, descending=True, stable=True)[:, case["top_groups"]:]
            out = torch.zeros_like(best).scatter_(1, worse, 1.0).repeat_interleave(e // case["groups"], 1)
            rank = torch.where(out > 0, -1e300, rank)
        at = rank.argsort(dim=1, descending=True, stable=True)[:, :k]
        at = torch.where(rank.gather(1, at) > -1e299, at, -1)
    picked = torch.where(at >= 0, score.gather(1, at.clamp(min=0)), 0.0)
    total = picked.sum(1, keepdim=True) if case["renormalise"] else torch.ones((t, 1), dtype=torch.float64, device="cuda")
    weights = torch.where(total > 0, picked / total, 0.0)
    if not case["back"]:
        return {"ids": None, "weights": weights, "offsets": None, "order": None, "position": None}
    dw = torch.where((at >= 0) & (total > 0), s["dweights"].double(), 0.0)
    slope = dw - (dw * weights).sum(1, keepdim=True) if case["renormalise"] else dw
    dscore = torch.zeros_like(score)
    dscore.scatter_add_(1, at.clamp(min=0), torch.where((at >= 0) & (total > 0), slope / total, 0.0))
    if case["score"] == "softmax":
        return {"dlogits": score * dscore - score * (score * dscore).sum(1, keepdim=True)}
    return {"dlogits": dscore * score * (-logits).sigmoid()}


def _exact_combine(case, s):
    t, k, w = (case[n] for n in ("tokens", "top_k", "width"))
    rows, at = s["rows"], s["position"].long()
    if not case["back"]:
        out = torch.zeros((t, w), dtype=torch.float64, device="cuda")
        for j in range(k):
            out += rows[at[:, j]].double() * s["weights"][:, j, None].double()
        return {"out": out}
    drows = torch.empty((t * k, w), dtype=torch.float64, device="cuda")
    dweights = torch.empty((t, k), dtype=torch.float64, device="cuda")
    for j in range(k):
        drows[at[:, j]] = s["dout"].double() * s["weights"][:, j, None].double()
        dweights[:, j] = (s["dout"].double() * rows[at[:, j]].double()).sum(1)
    return {"drows": drows, "dweights": dweights}
