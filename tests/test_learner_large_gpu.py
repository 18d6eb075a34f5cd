"""The learner layers over more than 2^31 elements, on streams of their own, and from two host threads."""
from __future__ import annotations

import threading

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _work(need):
    return torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def _big(gen, *shape):
    """bf16 noise without a wide intermediate."""
    v = torch.empty(shape, dtype=BF, device="cuda")
    for part in v.split(max(1, shape[0] // 16)):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda"))
    return v


@pytest.fixture(autouse=True)
def _room():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(3, 11_200_000, 64, 8), (132_000, 256, 64, 8)], ids=str)
def test_group_norm_over_2_31_elements(shape):
    """Every sample is computed alike, so the last ones have the bits that they have in a call of their own."""
    n, p, c, g = shape
    few = min(n, 2)
    x = _big(_gen(1), n, p, c)
    one = lambda k: tb.GroupNormDesc(samples=k, positions=p, channels=c, groups=g, type=1, activation=2, epsilon=1e-5)  # noqa: E731
    y, work = torch.empty_like(x), _work(tb.tb_cuda_group_norm_workspace(one(n)))
    mean, rstd = torch.empty((2, n, g), device="cuda")
    assert tb.tb_cuda_group_norm_device(one(n), x, None, None, y, mean, rstd, work) == 1
    tail = torch.empty_like(y[-few:])
    mean2, rstd2 = torch.empty((2, few, g), device="cuda")
    assert tb.tb_cuda_group_norm_device(one(few), x[-few:].clone(), None, None, tail, mean2, rstd2, work) == 1
    torch.cuda.synchronize()
    assert torch.equal(y[-few:], tail) and torch.equal(mean[-few:], mean2) and torch.equal(rstd[-few:], rstd2)
    # backward, dx over dy
    assert tb.tb_cuda_group_norm_backward_device(one(few), x[-few:].clone(), None, None, mean2, rstd2, tail, tail, None, None,
                                                 work) == 1
    assert tb.tb_cuda_group_norm_backward_device(one(n), x, None, None, mean, rstd, y, y, None, None, work) == 1
    torch.cuda.synchronize()
    assert torch.equal(y[-few:], tail)


@pytest.mark.parametrize("shape", [(33_000, 512, 128), (5, 3_400_000, 128), (2_200_000, 8, 128)], ids=str)
def test_gated_recurrence_over_2_31_elements(shape):
    """The last sequences agree with a call of their own: both lie within f32 sums of the definition, then one rounding
    to bf16 each."""
    b, t, d = shape
    few = 2
    gen = _gen(2)
    x, rec, inp = (_big(gen, b, t, d) for _ in range(3))
    decay, state = torch.linspace(-6.0, -3.0, d, device="cuda"), torch.randn((b, d), generator=gen, device="cuda")

    def run(k, x, rec, inp, state):
        desc = tb.GatedRecurrenceDesc(sequences=k, steps=t, channels=d, type=1, decay_scale=8.0)
        work = _work(tb.tb_cuda_gated_recurrence_workspace(desc))
        h, out = torch.empty_like(x), torch.empty_like(state)
        saved = torch.empty((k, -(-t // 16), d), device="cuda")
        assert tb.tb_cuda_gated_recurrence_device(desc, x, rec, inp, decay, None, None, state, h, out, saved, work) == 1
        torch.cuda.synchronize()
        keep = h[-few:].clone(), out[-few:].clone()
        dx, drec, dinp = h, torch.empty_like(h), torch.empty_like(h)  # the gradients may take h's place
        dh = x
        assert tb.tb_cuda_gated_recurrence_backward_device(desc, x.clone(), rec, inp, decay, None, None, saved, dh, None, dx,
                                                           drec, dinp, None, None, work) == 1
        torch.cuda.synchronize()
        return [v.float() for v in (*keep, dx[-few:], drec[-few:], dinp[-few:])]

    want = run(few, *(v[-few:].clone() for v in (x, rec, inp, state)))
    got = run(b, x, rec, inp, state)
    for a, v in zip(want, got):
        assert ((a - v).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -12 * a.abs().amax()).all()


def test_combine_over_2_31_elements():
    t, k, w = 700_000, 3, 1032
    gen = _gen(3)
    rows = _big(gen, t * k, w)
    position = torch.arange(t * k, dtype=torch.int32, device="cuda").reshape(t, k).flip(1).contiguous()
    weights = torch.rand((t, k), generator=gen, device="cuda")
    desc = lambda n: tb.ExpertCombineDesc(tokens=n, rows=n * k, width=w, top_k=k, type=1)  # noqa: E731
    out, few = torch.empty((t, w), dtype=BF, device="cuda"), 5
    assert tb.tb_cuda_combine_experts_device(desc(t), rows, position, weights, out) == 1
    tail = torch.empty((few, w), dtype=BF, device="cuda")
    last = position[-few:] - (t - few) * k
    assert tb.tb_cuda_combine_experts_device(desc(few), rows[-few * k:].clone(), last, weights[-few:].clone(), tail) == 1
    torch.cuda.synchronize()
    assert torch.equal(out[-few:], tail)
    drows, dweights = torch.empty_like(rows), torch.empty_like(weights)
    assert tb.tb_cuda_combine_experts_backward_device(desc(t), rows, position, weights, out, drows, dweights) == 1
    drows2, dweights2 = torch.empty_like(rows[-few * k:]), torch.empty((few, k), device="cuda")
    assert tb.tb_cuda_combine_experts_backward_device(desc(few), rows[-few * k:].clone(), last, weights[-few:].clone(), tail,
                                                      drows2, dweights2) == 1
    torch.cuda.synchronize()
    assert torch.equal(drows[-few * k:], drows2) and torch.equal(dweights[-few:], dweights2)


def test_route_over_2_31_elements():
    t, e, k = 2_150_000, 1000, 2
    gen = _gen(4)
    logits = _big(gen, t, e)
    desc = lambda n: tb.ExpertRouteDesc(tokens=n, experts=e, top_k=k, groups=1, top_groups=1, group_best=1, type=1,  # noqa: E731
                                        score=0, renormalise=0, weight_scale=1.0)
    whole = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731

    def run(n, logits):
        ids, weights = whole(n, k), torch.empty((n, k), device="cuda")
        offsets, order, position = whole(e + 1), whole(n * k), whole(n, k)
        assert tb.tb_cuda_route_experts_device(desc(n), logits, None, ids, weights, offsets, order, position,
                                               _work(tb.tb_cuda_route_experts_workspace(desc(n)))) == 1
        torch.cuda.synchronize()
        return ids, weights, offsets, order, position

    few = 100
    ids, weights, offsets, order, position = run(t, logits)
    ids2, weights2, *_ = run(few, logits[-few:].clone())
    assert torch.equal(ids[-few:], ids2) and torch.equal(weights[-few:], weights2)
    counts = torch.bincount(ids.flatten().long(), minlength=e)
    assert torch.equal(offsets.long().diff(), counts) and int(offsets[0]) == 0
    flat = torch.arange(t * k, device="cuda")
    assert torch.equal(order[position.flatten().long()].long(), flat)
    expert = ids.flatten().long()[order.long()]
    assert bool((expert.diff() >= 0).all()) and bool((order.long().diff()[expert.diff() == 0] > 0).all())
    dlogits, dw = torch.empty_like(logits), torch.randn((t, k), generator=gen, device="cuda")
    assert tb.tb_cuda_route_experts_backward_device(desc(t), logits, ids, dw, dlogits) == 1
    tail = torch.empty_like(logits[-few:])
    assert tb.tb_cuda_route_experts_backward_device(desc(few), logits[-few:].clone(), ids2, dw[-few:].clone(), tail) == 1
    torch.cuda.synchronize()
    assert torch.equal(dlogits[-few:], tail)


# ---- streams and threads ----

def _step(seed, scale):
    """Calls of every kind on tensors and workspaces of their own; returns what issues them on a stream, and the outputs."""
    gen = _gen(seed)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    whole = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    n, p, c, g = 6, 700 * scale, 64, 8
    norm = tb.GroupNormDesc(samples=n, positions=p, channels=c, groups=g, type=0, activation=2, epsilon=1e-5)
    x, dy, y, dx = new(n, p, c), new(n, p, c), new(n, p, c), new(n, p, c)
    mean, rstd, dgamma, dbeta = new(n, g), new(n, g), new(c), new(c)
    b, t, d = 4, 900 * scale, 40
    rec = tb.GatedRecurrenceDesc(sequences=b, steps=t, channels=d, type=0, decay_scale=8.0)
    seq, decay, state = [new(b, t, d) for _ in range(4)], new(d) - 3, new(b, d)
    h, out, saved, grads, ddecay = new(b, t, d), new(b, d), new(b, -(-t // 16), d), [new(b, t, d) for _ in range(3)], new(d)
    tok, e, k = 2000 * scale, 300, 5
    route = tb.ExpertRouteDesc(tokens=tok, experts=e, top_k=k, groups=10, top_groups=4, group_best=2, type=0, score=1,
                               renormalise=1, weight_scale=1.0)
    logits, bias = new(tok, e), new(e) * 0.01
    ids, weights, offsets, order, position = whole(tok, k), new(tok, k), whole(e + 1), whole(tok * k), whole(tok, k)
    works = [_work(tb.tb_cuda_group_norm_workspace(norm)), _work(tb.tb_cuda_gated_recurrence_workspace(rec)),
             _work(tb.tb_cuda_route_experts_workspace(route))]

    def issue(stream):
        return [tb.tb_cuda_group_norm_device(norm, x, None, None, y, mean, rstd, works[0], stream),
                tb.tb_cuda_group_norm_backward_device(norm, x, None, None, mean, rstd, dy, dx, dgamma, dbeta, works[0], stream),
                tb.tb_cuda_gated_recurrence_device(rec, *seq[:3], decay, None, None, state, h, out, saved, works[1], stream),
                tb.tb_cuda_gated_recurrence_backward_device(rec, *seq[:3], decay, None, None, saved, seq[3], out, *grads,
                                                            ddecay, None, works[1], stream),
                tb.tb_cuda_route_experts_device(route, logits, bias, ids, weights, offsets, order, position, works[2], stream)]

    return issue, [y, mean, rstd, dx, dgamma, dbeta, h, out, saved, *grads, ddecay, ids, weights, offsets, order, position]


def test_streams_with_workspaces_of_their_own():
    """Two programs' calls under way together give the bits that each gives alone."""
    steps = [_step(5, 3), _step(6, 1)]
    alone = []
    for issue, outputs in steps:
        assert all(issue(None))
        torch.cuda.synchronize()
        alone.append([v.clone() for v in outputs])
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for _, outputs in steps:
            for v in outputs:
                v.zero_()
        torch.cuda.synchronize()
        for (issue, _), stream in zip(steps, streams):
            assert all(issue(stream))
        torch.cuda.synchronize()
        for (_, outputs), want in zip(steps, alone):
            assert all(torch.equal(a, w) for a, w in zip(outputs, want))


def test_host_threads():
    """Four threads that call with other sizes at the same time, each on a stream of its own."""
    torch.cuda.init()
    steps = [_step(7 + i, 1 + i) for i in range(4)]
    alone = []
    for issue, outputs in steps:
        assert all(issue(None))
        torch.cuda.synchronize()
        alone.append([v.clone() for v in outputs])
    refused, ready = [], threading.Barrier(len(steps))

    def work(issue, stream):
        torch.cuda.set_device(0)
        ready.wait()
        for _ in range(20):
            refused.extend(v for v in issue(stream) if v != 1)

    threads = [threading.Thread(target=work, args=(issue, torch.cuda.Stream())) for issue, _ in steps]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not refused
    for (_, outputs), want in zip(steps, alone):
        assert all(torch.equal(a, w) for a, w in zip(outputs, want))
