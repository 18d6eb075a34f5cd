"""The routed experts' operators as workloads: tokens handed out to their experts, the experts' products, the same in
8-bit integers, and the orthogonalised update of their matrices, each in a plain form of elementary torch operations
and through this package's entry points.

The router lists the slots of each expert and the combine brings the experts' rows back; the operators below are what
lies between the two, at acting size (some aircraft, one step) and at training size (whole trajectories), and what an
optimiser does to the experts' matrices with their gradients."""
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
QUINTIC = (3.4445, -4.7750, 2.0315)  # the odd polynomial that drives every singular value to about 1
EPSILON = 1e-7


def listed():
    return [
        # acting: the slots of 61 aircraft, six experts each, weights applied on the way out
        dict(name="hand_out_act", op="hand", back=False, tokens=61, top_k=6, width=520, weights=True, masked=0.0,
             type="f32"),
        # training: the gradient of handing out, rows back to tokens and one number per slot
        dict(name="hand_out_train_backward", op="hand", back=True, tokens=16384, top_k=8, width=1024, weights=True,
             masked=0.1, type="bf16"),
        # acting: the same 61 aircraft's 366 rows through 64 experts; the weights are most of what is read
        dict(name="product_act", op="product", back=False, rows=366, used=366, experts=64, n_in=1024, n_out=2048,
             order="out_in", pad=0, type="bf16"),
        # training: the up projection of 16,384 steps, eight experts each
        dict(name="product_train", op="product", back=False, rows=131072, used=131072, experts=64, n_in=1024,
             n_out=2048, order="in_out", pad=0, type="bf16"),
        # training: both gradients of the down projection of half of them, a twentieth of the rows without a slot
        dict(name="product_train_backward", op="product", back=True, rows=65536, used=62259, experts=64, n_in=2048,
             n_out=1024, order="in_out", pad=0, type="bf16"),
        # a small learner in f32 on the library's inputs: 91 values and 4 views of 32 channels, odd rows
        dict(name="product_odd_f32_backward", op="product", back=True, rows=5003, used=5003, experts=12, n_in=219,
             n_out=384, order="in_out", pad=0, type="f32"),
        # acting: one aircraft through a dense layer with 8-bit weights
        dict(name="i8_act_single", op="i8", rows=1, used=1, experts=1, n_in=4096, n_out=4096, type="bf16"),
        # acting: 61 aircraft, 366 rows, 8-bit experts
        dict(name="i8_act_experts", op="i8", rows=366, used=366, experts=64, n_in=1024, n_out=2048, type="bf16"),
        # rollouts: a large batch through a dense 8-bit layer
        dict(name="i8_rollouts", op="i8", rows=16384, used=16384, experts=1, n_in=4096, n_out=4096, type="bf16"),
        # the small learner's eight experts
        dict(name="orthogonal_small", op="orthogonal", matrices=8, rows=128, columns=256, pad=0, type="f32"),
        # one odd dense matrix, taller than wide
        dict(name="orthogonal_odd", op="orthogonal", matrices=1, rows=2501, columns=1537, pad=3, type="f32"),
        # 64 experts' up projections
        dict(name="orthogonal_experts", op="orthogonal", matrices=64, rows=1024, columns=2048, pad=0, type="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def _width(rng, low, high):
    """Any width, or one that is a multiple of 64."""
    return _spread(rng, low, high) if rng.random() < 0.4 else 64 * _spread(rng, 1, high // 64)


def draw(rng):
    op = rng.choice(["hand", "product", "product", "i8", "orthogonal"])
    kind = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "hand":
        top_k, width = rng.randint(1, 12), _width(rng, 1, 2048)
        return dict(op=op, back=rng.random() < 0.5, tokens=_spread(rng, 1, max(1, min(65536, 60_000_000 // (top_k * width)))),
                    top_k=top_k, width=width, weights=rng.random() < 0.6, masked=rng.choice([0.0, 0.2]), type=kind)
    if op == "orthogonal":
        rows, columns = _width(rng, 2, 2048), _width(rng, 2, 2048)
        small = min(rows, columns)
        most = 2_000_000_000_000 // (5 * 3 * small * rows * columns)
        return dict(op=op, matrices=_spread(rng, 1, max(1, min(64, most))), rows=rows, columns=columns,
                    pad=rng.choice([0, 0, 8, 1]), type=kind)
    experts = rng.choice([1, _spread(rng, 2, 128)])
    n_in, n_out = _width(rng, 8, 4096), _width(rng, 8, 4096)
    while experts * n_in * n_out > 100_000_000:
        experts = -(-experts // 2)
        n_in, n_out = -(-n_in // 2), -(-n_out // 2)
    rows = _spread(rng, 1, max(1, min(131072, 60_000_000_000 // (n_in * n_out), 100_000_000 // (n_in + n_out))))
    used = rows if rng.random() < 0.7 else rng.randint(1, rows)
    case = dict(op=op, rows=rows, used=used, experts=experts, n_in=n_in, n_out=n_out, type=kind)
    if op == "product":
        case.update(back=rng.random() < 0.5, order=rng.choice(["in_out", "out_in"]), pad=rng.choice([0, 0, 8, 3]))
    return case


# ---- inputs ----

def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"hand": _prepare_hand, "product": _prepare_product, "i8": _prepare_i8,
             "orthogonal": _prepare_orthogonal}[case["op"]](case, gen)
    state["case"] = case
    if own:  # what a user's program keeps between calls: the descriptor, the workspace and the output buffers
        _plan(case, state)
    return state


def _prepare_hand(case, gen):
    t, k, w = (case[n] for n in ("tokens", "top_k", "width"))
    kind = TYPES[case["type"]]
    # slots sorted by expert: any order of those that have one; masked tokens' slots have none
    free = torch.rand((t,), generator=gen, device="cuda") >= case["masked"]
    slots = torch.randperm(t * k, generator=gen, device="cuda")
    order = torch.cat([slots[free[slots // k]], torch.full((t * k,), -1, device="cuda")])[:t * k]
    position = torch.full((t * k + 1,), -1, device="cuda")
    position[order.where(order >= 0, t * k)] = torch.arange(t * k, device="cuda")
    position = position[:-1].masked_fill(~free.repeat_interleave(k), -1)
    s = {"order": order.to(torch.int32), "position": position.reshape(t, k).to(torch.int32),
         "x": _normal((t, w), gen).to(kind), "weights": None, "rows": torch.zeros((t * k, w), dtype=kind, device="cuda")}
    if case["weights"]:
        s["weights"] = torch.rand((t, k), generator=gen, device="cuda")
    if case["back"]:
        s["drows"] = _normal((t * k, w), gen).to(kind)
    return s


def _offsets(case, gen):
    """Each expert's rows: some experts are busier than others, and few rows leave some with none."""
    e, used = case["experts"], case["used"]
    busy = torch.softmax(_normal((e,), gen, 0.5), 0)
    edges = torch.cat([busy.cumsum(0)[:-1], torch.full((1,), 2.0, device="cuda")])
    owner = torch.bucketize(torch.rand((used,), generator=gen, device="cuda"), edges)
    count = torch.bincount(owner, minlength=e)
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), count.cumsum(0)]).to(torch.int32), int(count.max())


def _prepare_product(case, gen):
    r, e, n, m, pad = (case[k] for k in ("rows", "experts", "n_in", "n_out", "pad"))
    kind = TYPES[case["type"]]
    offsets, most = _offsets(case, gen)
    shape = (e, n, m) if case["order"] == "in_out" else (e, m, n)
    s = {"offsets": offsets, "most": most, "w": _normal(shape, gen, n ** -0.5).to(kind),
         # `pad` > 0: the rows are slices of wider ones
         "x": _normal((r, n + pad), gen).to(kind)[:, :n], "y": torch.zeros((r, m), dtype=kind, device="cuda")}
    if case["back"]:
        s["dy"] = _normal((r, m), gen).to(kind)
        s["dx"], s["dw"] = torch.zeros((r, n), dtype=kind, device="cuda"), torch.zeros_like(s["w"])
    return s


def _prepare_i8(case, gen):
    r, e, n, m = (case[k] for k in ("rows", "experts", "n_in", "n_out"))
    kind = TYPES[case["type"]]
    offsets, most = _offsets(case, gen)
    w = _normal((e, m, n), gen, n ** -0.5)
    scale = w.abs().amax(2) / 127
    return {"offsets": offsets, "most": most, "x": _normal((r, n), gen).to(kind), "w_scale": scale,
            "w": torch.round(w / scale[..., None]).to(torch.int8), "y": torch.zeros((r, m), dtype=kind, device="cuda")}


def _prepare_orthogonal(case, gen):
    b, m, n, pad = (case[k] for k in ("matrices", "rows", "columns", "pad"))
    # a gradient's shape: noise, and directions that fall off in strength
    g = _normal((b, m, n + pad), gen)
    rank = min(8, m, n)
    strength = 4.0 * (m + n) ** 0.5 * 0.6 ** torch.arange(rank, device="cuda")
    u, v = _normal((b, m, rank), gen, m ** -0.5), _normal((b, rank, n + pad), gen, n ** -0.5)
    return {"g": ((g + (u * strength) @ v) * 1e-3).to(TYPES[case["type"]])[..., :n]}


# ---- the work that no form can do without ----

def work(case):
    s = SIZE[case["type"]]
    if case["op"] == "hand":
        n, slots = case["tokens"] * case["width"], case["tokens"] * case["top_k"]
        moved = n * case["top_k"] * s + 4 * slots * (1 + case["weights"])
        if case["back"]:
            return {"bytes": 2 * n * s + moved + 4 * slots * case["weights"], "flops": 4 * n * case["top_k"]}
        return {"bytes": n * s + moved, "flops": n * case["top_k"]}
    if case["op"] == "orthogonal":
        n = case["matrices"] * case["rows"] * case["columns"]
        small = min(case["rows"], case["columns"])
        # a symmetric product is half of a product
        return {"bytes": 2 * n * s, "flops": 5 * (3 * n * small + case["matrices"] * small ** 3)}
    r, n, m = case["used"], case["n_in"], case["n_out"]
    weights = min(case["experts"], r) * n * m
    if case["op"] == "i8":
        return {"bytes": weights + r * (n + m) * s, "flops": 2 * r * n * m}
    if case["back"]:
        return {"bytes": (weights + case["experts"] * n * m + r * (2 * n + m)) * s, "flops": 4 * r * n * m}
    return {"bytes": (weights + r * (n + m)) * s, "flops": 2 * r * n * m}


# ---- one pass ----

def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"], case.get("back", False)](state)
    return _PLAIN[case["op"], case.get("back", False)](case, state)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end ----

def _plain_hand(case, s):
    slot = s["order"].long()
    there = (slot >= 0)[:, None]
    slot = slot.clamp(min=0)
    rows = s["x"].float()[slot // case["top_k"]]
    if s["weights"] is not None:
        rows = rows * s["weights"].flatten()[slot][:, None]
    return {"rows": torch.where(there, rows, 0 * rows).to(s["x"].dtype)}


def _plain_hand_back(case, s):
    there = (s["position"] >= 0)[..., None]
    back = torch.where(there, s["drows"].float()[s["position"].clamp(min=0).long()], torch.zeros((), device="cuda"))
    x = s["x"].float()
    if s["weights"] is None:
        return {"dx": back.sum(1).to(s["x"].dtype)}
    return {"dx": (back * s["weights"][..., None]).sum(1).to(s["x"].dtype), "dweights": (back * x[:, None]).sum(2)}


def _places(case, s):
    """Each expert's rows side by side, padded to the busiest one's: [experts, most] rows, and which of them are."""
    at = s["offsets"][:-1, None].long() + torch.arange(s["most"], device="cuda")
    there = at < s["offsets"][1:, None]
    return at.clamp(max=case["rows"] - 1), there


def _padded(v, at, there):
    return torch.where(there[..., None], v.float()[at], torch.zeros((), device="cuda"))


def _unpadded(v, at, there, rows):
    out = torch.zeros((rows + 1, v.shape[2]), device="cuda")
    out[torch.where(there, at, rows).flatten()] = v.flatten(0, 1)
    return out[:rows]


def _plain_product(case, s):
    at, there = _places(case, s)
    w = s["w"].float() if case["order"] == "in_out" else s["w"].float().transpose(1, 2)
    y = torch.bmm(_padded(s["x"], at, there), w)
    return {"y": _unpadded(y, at, there, case["rows"]).to(s["x"].dtype)}


def _plain_product_back(case, s):
    at, there = _places(case, s)
    kind = s["x"].dtype
    w = s["w"].float() if case["order"] == "out_in" else s["w"].float().transpose(1, 2)
    x, dy = _padded(s["x"], at, there), _padded(s["dy"], at, there)
    dx = _unpadded(torch.bmm(dy, w), at, there, case["rows"])
    left, right = (x, dy) if case["order"] == "in_out" else (dy, x)
    return {"dx": dx.to(kind), "dw": torch.bmm(left.transpose(1, 2), right).to(kind)}


def _plain_i8(case, s):
    x = s["x"].float()
    most = x.abs().amax(1)
    q = torch.round(x * (127 / most)[:, None])
    scale = most / 127
    at, there = _places(case, s)
    y = torch.bmm(_padded(q, at, there), s["w"].float().transpose(1, 2)) * scale[at][..., None] * s["w_scale"][:, None]
    return {"y": _unpadded(y, at, there, case["rows"]).to(s["x"].dtype), "scale": scale}


def _quintic(x):
    a, b, c = QUINTIC
    square = torch.bmm(x, x.transpose(1, 2))
    return a * x + torch.bmm(b * square + c * torch.bmm(square, square), x)


def _plain_orthogonal(case, s):
    g = s["g"].float()
    if case["rows"] > case["columns"]:
        g = g.transpose(1, 2)
    x = g / (torch.sqrt((g * g).sum((1, 2), keepdim=True)) + EPSILON)
    x = _quintic(_quintic(_quintic(_quintic(_quintic(x)))))
    return {"update": (x.transpose(1, 2) if case["rows"] > case["columns"] else x).to(s["g"].dtype)}


_PLAIN = {("hand", False): _plain_hand, ("hand", True): _plain_hand_back, ("product", False): _plain_product,
          ("product", True): _plain_product_back, ("i8", False): _plain_i8, ("orthogonal", False): _plain_orthogonal}


# ---- the definitions in 64 bits, expert by expert and matrix by matrix ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "hand":
        return _exact_hand(case, s)
    if case["op"] == "orthogonal":
        return {"update": torch.stack([_exact_update(g) for g in s["g"].double()])}
    ends = s["offsets"].tolist()
    spans = [(e, slice(a, z)) for e, (a, z) in enumerate(zip(ends, ends[1:])) if z > a]
    if case["op"] == "i8":
        x = s["x"].double()
        scale = x.abs().amax(1) / 127
        q = torch.round(x / scale[:, None]) * scale[:, None]
        y = torch.zeros_like(s["y"], dtype=torch.float64)
        for e, rows in spans:
            y[rows] = q[rows] @ (s["w"][e].double() * s["w_scale"][e].double()[:, None]).T
        return {"y": y, "scale": scale}
    x, turned = s["x"].double(), case["order"] == "out_in"
    if not case["back"]:
        y = torch.zeros_like(s["y"], dtype=torch.float64)
        for e, rows in spans:
            y[rows] = x[rows] @ (s["w"][e].double().T if turned else s["w"][e].double())
        return {"y": y}
    dy, dx, dw = s["dy"].double(), torch.zeros_like(x), torch.zeros_like(s["w"], dtype=torch.float64)
    for e, rows in spans:
        dx[rows] = dy[rows] @ (s["w"][e].double() if turned else s["w"][e].double().T)
        dw[e] = dy[rows].T @ x[rows] if turned else x[rows].T @ dy[rows]
    return {"dx": dx, "dw": dw}


def _exact_hand(case, s):
    x, k = s["x"].double(), case["top_k"]
    weights = torch.ones(s["position"].shape, dtype=torch.float64, device="cuda") if s["weights"] is None else s["weights"].double()
    if not case["back"]:
        rows = torch.zeros_like(s["rows"], dtype=torch.float64)
        for j in range(k):
            has = s["position"][:, j] >= 0
            rows[s["position"][has, j].long()] = x[has] * weights[has, j, None]
        return {"rows": rows}
    dx, dweights = torch.zeros_like(x), torch.zeros_like(weights)
    for j in range(k):
        has = s["position"][:, j] >= 0
        back = s["drows"][s["position"][has, j].long()].double()
        dx[has] += back * weights[has, j, None]
        dweights[has, j] = torch.einsum("tw,tw->t", back, x[has])
    return {"dx": dx} if s["weights"] is None else {"dx": dx, "dweights": dweights}


def _exact_update(g):
    """The polynomial, five times, on the smaller side's Gram matrix."""
    a, b, c = QUINTIC
    wide = g if g.shape[0] <= g.shape[1] else g.T
    x = wide / (torch.linalg.matrix_norm(wide) + EPSILON)
    for _ in range(5):
        gram = x @ x.T
        x = (a * torch.eye(gram.shape[0], dtype=g.dtype, device=g.device) + b * gram + c * (gram @ gram)) @ x
    return x if g.shape[0] <= g.shape[1] else x.T


# ---- the same through the package ----

def _tb():
    import turbinator_c_b200
    return turbinator_c_b200


def _type(case):
    tb = _tb()
    return {"f32": tb.TB_TYPE_F32, "bf16": tb.TB_TYPE_BF16, "f16": tb.TB_TYPE_F16}[case["type"]]


def _scratch(need):
    return torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")


def _plan(case, s):
    tb = _tb()
    if case["op"] == "hand":
        s["desc"] = tb.ExpertCombineDesc(tokens=case["tokens"], rows=case["tokens"] * case["top_k"], width=case["width"],
                                         top_k=case["top_k"], type=_type(case))
        s["dx"] = torch.empty_like(s["x"])
        s["dweights"] = None if s["weights"] is None else torch.empty_like(s["weights"])
    elif case["op"] == "product":
        s["desc"] = tb.ExpertProductDesc(
            rows=case["rows"], experts=case["experts"], in_width=case["n_in"], out_width=case["n_out"],
            in_stride=case["n_in"] + case["pad"], din_stride=case["n_in"], type=_type(case),
            weight_order=tb.TB_WEIGHT_IN_OUT if case["order"] == "in_out" else tb.TB_WEIGHT_OUT_IN)
        s["work"] = _scratch(tb.tb_cuda_experts_product_workspace(s["desc"]))
    elif case["op"] == "i8":
        s["quantise"] = tb.QuantiseDesc(rows=case["rows"], width=case["n_in"], type=_type(case))
        s["desc"] = tb.ExpertProductI8Desc(rows=case["rows"], experts=case["experts"], in_width=case["n_in"],
                                           out_width=case["n_out"], type=_type(case))
        s["work"] = _scratch(tb.tb_cuda_experts_product_i8_workspace(s["desc"]))
        s["q"] = torch.empty((case["rows"], case["n_in"]), dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(case["rows"], device="cuda")
    else:
        a, b, c = QUINTIC
        stride = case["columns"] + case["pad"]
        s["desc"] = tb.OrthogonaliseDesc(matrices=case["matrices"], rows=case["rows"], columns=case["columns"],
                                         in_matrix_stride=case["rows"] * stride, in_row_stride=stride, steps=5, a=a, b=b,
                                         c=c, epsilon=EPSILON, scale=1.0, type=_type(case))
        s["work"] = _scratch(tb.tb_cuda_orthogonalise_workspace(s["desc"]))
        s["update"] = torch.empty(s["g"].shape, dtype=s["g"].dtype, device="cuda")


def _call(ok):
    if ok != 1:
        raise RuntimeError("the call was refused")


def _own_hand(s):
    _call(_tb().tb_cuda_hand_out_experts_device(s["desc"], s["x"], s["order"], s["weights"], s["rows"],
                                                torch.cuda.current_stream()))
    return {"rows": s["rows"]}


def _own_hand_back(s):
    _call(_tb().tb_cuda_hand_out_experts_backward_device(s["desc"], s["x"], s["position"], s["weights"], s["drows"],
                                                         s["dx"], s["dweights"], torch.cuda.current_stream()))
    return {"dx": s["dx"]} if s["weights"] is None else {"dx": s["dx"], "dweights": s["dweights"]}


def _own_product(s):
    _call(_tb().tb_cuda_experts_product_device(s["desc"], s["x"], s["w"], s["offsets"], s["y"], s["work"],
                                               torch.cuda.current_stream()))
    return {"y": s["y"]}


def _own_product_back(s):
    _call(_tb().tb_cuda_experts_product_backward_device(s["desc"], s["x"], s["w"], s["offsets"], s["dy"], s["dx"], s["dw"],
                                                        s["work"], torch.cuda.current_stream()))
    return {"dx": s["dx"], "dw": s["dw"]}


def _own_i8(s):
    tb, stream = _tb(), torch.cuda.current_stream()
    _call(tb.tb_cuda_quantise_rows_device(s["quantise"], s["x"], s["q"], s["scale"], stream))
    _call(tb.tb_cuda_experts_product_i8_device(s["desc"], s["q"], s["scale"], s["w"], s["w_scale"], s["offsets"], s["y"],
                                               s["work"], stream))
    return {"y": s["y"], "scale": s["scale"]}


def _own_orthogonal(s):
    _call(_tb().tb_cuda_orthogonalise_device(s["desc"], s["g"], s["update"], s["work"], torch.cuda.current_stream()))
    return {"update": s["update"]}


_OWN = {("hand", False): _own_hand, ("hand", True): _own_hand_back, ("product", False): _own_product,
        ("product", True): _own_product_back, ("i8", False): _own_i8, ("orthogonal", False): _own_orthogonal}
