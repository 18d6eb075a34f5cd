"""The learner layers together: the example's training and acting, capture into a CUDA graph, and corners of the
selection that random logits seldom reach."""
from __future__ import annotations

import importlib.util
import os

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("learner_step", os.path.join(ROOT, "examples", "learner_step.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_learns_and_acts_as_it_was_trained(example):
    actor = example.Actor(dtype=torch.float32)
    losses = example.train(actor, aircraft=8, steps=20, updates=30)
    assert losses[-1] < 0.5 * losses[0], losses
    proprio, luma, reset = example.trajectories(3, 18, seed=1)
    with torch.no_grad():
        whole = actor(proprio, luma, torch.zeros((3, actor.width), device="cuda"), reset)[0]
    # two orders of the same sums in f32, through layers of a few hundred terms
    assert torch.allclose(example.act(actor, proprio, luma, reset), whole, rtol=1e-3, atol=1e-3)


def test_example_gradient_is_the_difference(example):
    """The loss's change along a random direction of all parameters, by the layers' gradients and by differences."""
    actor = example.Actor(width=32, experts=4, stem=16, dtype=torch.float32, seed=3)
    proprio, luma, reset = example.trajectories(4, 17, seed=2)
    first = torch.zeros((4, actor.width), device="cuda")

    def loss():
        guess, _, _ = actor(proprio[:, :-1], luma[:, :-1], first, reset[:, :-1].contiguous())
        return (guess - proprio[:, 1:]).double().square().mean()

    loss().backward()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    ways = [torch.randn(p.shape, generator=gen, device="cuda") * p.detach().abs().mean() for p in actor.parameters()]
    # a few tokens may change experts along the way: the router keeps its logits
    ways = [torch.zeros_like(w) if p is actor.router else w for p, w in zip(actor.parameters(), ways)]
    slope = sum(float((p.grad.double() * w.double()).sum()) for p, w in zip(actor.parameters(), ways))

    def at(step):
        with torch.no_grad():
            for p, w in zip(actor.parameters(), ways):
                p.add_(w, alpha=step)
            value = float(loss())
            for p, w in zip(actor.parameters(), ways):
                p.sub_(w, alpha=step)
        return value

    # the difference's own error: curvature (step^2) and f32 rounding of the loss (about 1e-6 / step)
    step = 2e-3
    assert abs((at(step) - at(-step)) / (2 * step) - slope) < 0.03 * abs(slope) + 2e-3


def test_layers_captured_in_a_cuda_graph():
    """A step of every layer, forward and backward, replays with the bits of the direct calls."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    new = lambda *s, kind=torch.float32: torch.randn(s, generator=gen, device="cuda").to(kind)  # noqa: E731
    bf = torch.bfloat16
    n, p, c, g = 12, 300, 64, 8
    norm = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=1, activation=2, epsilon=1e-5)
    x, dy, gamma, beta = new(n, p, c, kind=bf), new(n, p, c, kind=bf), new(c), new(c)
    y, dx, mean, rstd = torch.empty_like(x), torch.empty_like(x), new(n, g), new(n, g)
    dgamma, dbeta = new(c), new(c)
    b, t, d = 400, 300, 64  # many rounds: bulk copies; and strips, with three sequences
    long = tb.GatedRecurrenceDesc(sequences=b, steps=t, channels=d, type=1, decay_scale=8.0)
    few = tb.GatedRecurrenceDesc(sequences=3, steps=b * t // 3, channels=d, type=1, decay_scale=8.0)
    seq = [new(b, t, d, kind=bf) for _ in range(4)]
    decay, h = new(d) - 3, new(b, t, d, kind=bf)
    saved = [new(b, -(-t // 16), d), new(3, -(-(b * t // 3) // 16), d)]
    grads = [[torch.empty_like(h) for _ in range(3)] + [new(d)] for _ in range(2)]
    tok, e, k = 3000, 96, 4
    route = tb.ExpertRouteDesc(tokens=tok, experts=e, top_k=k, groups=1, top_groups=1, group_best=1, type=0, score=1,
                               renormalise=1, weight_scale=1.0)
    logits, bias, dw, dlogits = new(tok, e), new(e) * 0.01, new(tok, k), new(tok, e)
    whole = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, offsets, order, position, weights = whole(tok, k), whole(e + 1), whole(tok * k), whole(tok, k), new(tok, k)
    comb = tb.ExpertCombineDesc(tokens=tok, rows=tok * k, width=72, top_k=k, type=1)
    rows, out, dout = new(tok * k, 72, kind=bf), new(tok, 72, kind=bf), new(tok, 72, kind=bf)
    drows, dweights = torch.empty_like(rows), new(tok, k)
    need = max(tb.tb_cuda_group_norm_workspace(norm), tb.tb_cuda_gated_recurrence_workspace(long),
               tb.tb_cuda_gated_recurrence_workspace(few), tb.tb_cuda_route_experts_workspace(route))
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()

    def step():
        assert tb.tb_cuda_group_norm_device(norm, x, gamma, beta, y, mean, rstd, work, s) == 1
        assert tb.tb_cuda_group_norm_backward_device(norm, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta, work, s) == 1
        for desc, keep, grad in zip((long, few), saved, grads):
            assert tb.tb_cuda_gated_recurrence_device(desc, *seq[:3], decay, None, None, None, h, None, keep, work, s) == 1
            assert tb.tb_cuda_gated_recurrence_backward_device(desc, *seq[:3], decay, None, None, keep, seq[3], None,
                                                               *grad, None, work, s) == 1
        assert tb.tb_cuda_route_experts_device(route, logits, bias, ids, weights, offsets, order, position, work, s) == 1
        assert tb.tb_cuda_route_experts_backward_device(route, logits, ids, dw, dlogits, s) == 1
        assert tb.tb_cuda_combine_experts_device(comb, rows, position, weights, out, s) == 1
        assert tb.tb_cuda_combine_experts_backward_device(comb, rows, position, weights, dout, drows, dweights, s) == 1

    outputs = [y, dx, mean, rstd, dgamma, dbeta, h, *saved, *grads[0], *grads[1], ids, weights, offsets, order, position,
               dlogits, out, drows, dweights]
    torch.cuda.synchronize()
    step()
    s.synchronize()
    direct = [v.clone() for v in outputs]
    for v in outputs:
        v.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(direct, outputs))
    assert tb.tb_cuda_synchronize(s) == 1


@pytest.mark.parametrize("kind", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("experts", (64, 256, 512, 1000))
def test_route_best_experts_next_to_each_other(kind, experts):
    """All of a token's best experts in one run, wherever it starts, in any order of their logits, and with ties."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)
    t, k = 200, 12
    logits = torch.randn((t, experts), generator=gen, device="cuda").clamp(-3, 3)
    for i in range(t):
        first = (i * 7) % (experts - k - 4)
        run = torch.randperm(k + 4, generator=gen, device="cuda").float() * 0.25 + 5.0
        logits[i, first:first + k + 4] = 5.0 if i % 5 == 0 else run
    logits = logits.to(kind)
    desc = tb.ExpertRouteDesc(tokens=t, experts=experts, top_k=k, groups=1, top_groups=1, group_best=1,
                              type={torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[kind], score=0, renormalise=1,
                              weight_scale=1.0)
    ids, weights = torch.empty((t, k), dtype=torch.int32, device="cuda"), torch.empty((t, k), device="cuda")
    work = torch.empty(tb.tb_cuda_route_experts_workspace(desc), dtype=torch.uint8, device="cuda")
    assert tb.tb_cuda_route_experts_device(desc, logits, None, ids, weights, None, None, None, work) == 1
    torch.cuda.synchronize()
    want = logits.float().sort(dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(ids.long(), want)
    # with a bias (ranked by scores): the same experts where the bias is nothing and no two scores are alike
    zero = torch.zeros(experts, device="cuda")
    assert tb.tb_cuda_route_experts_device(desc, logits, zero, ids, weights, None, None, None, work) == 1
    torch.cuda.synchronize()
    distinct = torch.arange(t, device="cuda") % 5 != 0
    assert torch.equal(ids.long()[distinct], want[distinct])


def _routed(kind, logits, bias, top_k, score, groups=1):
    t, experts = logits.shape
    desc = tb.ExpertRouteDesc(tokens=t, experts=experts, top_k=top_k, groups=groups, top_groups=1, group_best=1,
                              type={torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[kind], score=score,
                              renormalise=1, weight_scale=1.0)
    whole = lambda *s: torch.full(s, -77, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, weights = whole(t, top_k), torch.full((t, top_k), float("nan"), device="cuda")
    offsets, order, position = whole(experts + 1), whole(t * top_k), whole(t, top_k)
    work = torch.empty(tb.tb_cuda_route_experts_workspace(desc), dtype=torch.uint8, device="cuda")
    assert tb.tb_cuda_route_experts_device(desc, logits, bias, ids, weights, offsets, order, position, work) == 1
    torch.cuda.synchronize()
    return ids.long(), weights, offsets.long()


@pytest.mark.parametrize("kind", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("experts", (256, 512, 1024))
@pytest.mark.parametrize("top_k", (5, 6, 8, 17, 32))
def test_route_takes_every_expert_that_is_there(kind, experts, top_k):
    """A token with few available experts, all in one run of experts/32 of them, gets all that it has slots for."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(8)
    run, t = experts // 32, 32 * (experts // 32)
    token = torch.arange(t, device="cuda")
    first, many = token % 32 * run, token // 32 + 1  # 1 .. run of them
    place = torch.rand((t, run), generator=gen, device="cuda").argsort(1)
    logits = torch.full((t, experts), float("-inf"), device="cuda")
    values = place.float() * 0.25 - 3.0  # distinct in every type, and so are their sigmoids
    chosen = torch.rand((t, run), generator=gen, device="cuda").argsort(1) < many[:, None]
    logits.scatter_(1, first[:, None] + torch.arange(run, device="cuda"),
                    torch.where(chosen, values, float("-inf")))
    logits = logits.to(kind)
    l64 = logits.double()
    want = l64.sort(dim=1, descending=True, stable=True)[1][:, :top_k]
    taken = torch.arange(top_k, device="cuda") < many.clamp(max=top_k)[:, None]
    want = torch.where(taken, want, -1)
    counts = torch.zeros(experts, dtype=torch.long, device="cuda").index_add_(0, want[taken], torch.ones_like(want[taken]))
    for score, bias in ((tb.TB_SCORE_SOFTMAX, None), (tb.TB_SCORE_SIGMOID, None),
                        (tb.TB_SCORE_SIGMOID, torch.zeros(experts, device="cuda"))):
        ids, weights, offsets = _routed(kind, logits, bias, top_k, score)
        assert torch.equal(ids, want)
        assert torch.equal(offsets.diff(), counts)
        picked = torch.where(taken, l64.gather(1, want.clamp(min=0)), float("-inf"))
        s = picked.softmax(1) if score == tb.TB_SCORE_SOFTMAX else torch.sigmoid(picked)
        # scores within 16 U, their sum of at most 32 terms within 48, one division
        assert ((weights.double() - s / s.sum(1, keepdim=True)).abs() <= 96 * 2.0 ** -24 * s / s.sum(1, keepdim=True)).all()


@pytest.mark.parametrize("kind", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("experts", (256, 512, 1024))
def test_route_takes_the_whole_of_a_group_in_one_run(kind, experts):
    """Groups of experts/32: all slots come from the token's one group."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    per, t = experts // 32, 96
    logits = (torch.rand((t, experts), generator=gen, device="cuda").argsort(1).float() / experts * 4 - 2)
    group = torch.arange(t, device="cuda") % 32
    inside = torch.arange(experts, device="cuda")[None] // per == group[:, None]
    logits = torch.where(inside, torch.rand((t, experts), generator=gen, device="cuda").argsort(1) * (1 / 128) + 3.0, logits)
    logits = logits.to(kind)
    want = logits.float().masked_fill(~inside, float("-inf")).sort(dim=1, descending=True, stable=True)[1][:, :min(per, 32)]
    for top_k in {5, 8, min(per, 32)}:
        ids, _, _ = _routed(kind, logits, None, top_k, tb.TB_SCORE_SOFTMAX, groups=32)
        assert torch.equal(ids, want[:, :top_k])


def test_example_reports_a_wait_that_ran_out(example, monkeypatch):
    """Training and acting end with an error where the stream's status says that a kernel gave up waiting."""
    actor = example.Actor(width=32, experts=4, stem=16, dtype=torch.float32)
    proprio, luma, reset = example.trajectories(2, 3)
    asked = []
    monkeypatch.setattr(tb, "tb_cuda_synchronize", lambda stream=None: asked.append(stream) or 0)
    with pytest.raises(RuntimeError, match="gave up waiting"):
        example.act(actor, proprio, luma, reset)
    with pytest.raises(RuntimeError, match="gave up waiting"):
        example.train(actor, aircraft=2, steps=3, updates=1)
    assert [s.cuda_stream for s in asked] == [torch.cuda.current_stream().cuda_stream] * 2


@pytest.mark.parametrize("score", (tb.TB_SCORE_SOFTMAX, tb.TB_SCORE_SIGMOID))
@pytest.mark.parametrize("experts,groups", ((40, 1), (64, 8), (300, 1)))
def test_route_bias_takes_experts_out(score, experts, groups):
    """No token gets an expert whose bias is -inf or NaN, and the others' lists are those of a call in which it is not
    available."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(10)
    t, k = 300, 4
    logits = torch.randn((t, experts), generator=gen, device="cuda")
    bias = torch.randint(-30, 31, (experts,), generator=gen, device="cuda") * 0.01
    out = torch.randperm(experts, generator=gen, device="cuda")[:experts // 3]
    gone = bias.clone()
    gone[out[::2]], gone[out[1::2]] = -float("inf"), float("nan")
    ids, weights, _ = _routed(torch.float32, logits, gone, k, score, groups)
    taken = ids >= 0
    assert not torch.isin(ids[taken], out).any()
    if score == tb.TB_SCORE_SIGMOID:  # whose scores do not depend on the others
        logits[:, out] = -float("inf")
        ids2, weights2, _ = _routed(torch.float32, logits, bias, k, score, groups)
        assert torch.equal(ids, ids2) and torch.equal(weights, weights2)
    if groups == 1:
        assert taken.all()


def test_route_near_ties_of_softmax_scores_with_a_bias():
    """Scores within a few roundings of each other, told apart by the bias alone or not at all: whichever comes first,
    the ranking values fall by no more than the stated error of a score, and none is left out that is clearly above."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    t, e, k = 500, 96, 7
    logits = torch.randint(-8, 1, (t, e), generator=gen, device="cuda") * 0.5
    logits += torch.randint(-3, 4, (t, e), generator=gen, device="cuda") * 2.0 ** -21
    bias = torch.randint(-2, 3, (e,), generator=gen, device="cuda") * 2.0 ** -14
    ids, _, _ = _routed(torch.float32, logits, bias, k, tb.TB_SCORE_SOFTMAX)
    l64 = logits.double()
    rank = l64.softmax(1) + bias.double()
    spread = l64.amax(1, keepdim=True) - l64
    # a score's stated error, and the rounding of its sum with the bias
    error = (4 + spread) * 2.0 ** -20 * l64.softmax(1) + 2.0 ** -24 * rank.abs()
    assert int(ids.min()) >= 0 and all(len(set(r)) == k for r in ids.tolist())
    got, near = rank.gather(1, ids), error.gather(1, ids)
    assert (got[:, 1:] - got[:, :-1] <= near[:, 1:] + near[:, :-1]).all()
    rest = rank.scatter(1, ids, -float("inf"))
    worst = (got - near)[:, -1:]
    assert (rest - error.scatter(1, ids, 0.0) <= worst + 2 * near[:, -1:]).all()
