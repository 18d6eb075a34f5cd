"""The example with its experts' operators: it trains by orthogonalised momentum, acts with the experts in 8 bits, and the
gradients of its layers of experts are those of differences."""
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


@pytest.mark.parametrize("kind", (torch.float32, torch.bfloat16), ids=str)
def test_example_trains_by_orthogonalised_momentum_and_acts_in_8_bits(example, kind):
    actor = example.Actor(width=64, experts=4, stem=16, dtype=kind)
    before = actor.up.detach().clone()
    losses = example.train(actor, aircraft=4, steps=9, updates=3, orthogonal=True)
    assert all(v == v and abs(v) < 1e6 for v in losses)
    step = (actor.up.detach() - before).float()
    assert torch.isfinite(step).all() and (step.abs().amax((1, 2)) > 0).any()
    proprio, luma, reset = example.trajectories(3, 6, seed=1)
    plain = example.act(actor, proprio, luma, reset)
    actor.hold_experts_in_8_bits()
    held = example.act(actor, proprio, luma, reset)
    assert held.shape == plain.shape and torch.isfinite(held.float()).all()


def test_example_momentum_moves_every_direction_alike(example):
    """One step of a fresh momentum is rate x the orthogonalised gradient: singular values within those of the quintic."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    p = torch.nn.Parameter(torch.randn((2, 40, 60), generator=gen, device="cuda"))
    p.grad = torch.randn((2, 40, 60), generator=gen, device="cuda")
    before = p.detach().clone()
    example.OrthogonalMomentum([p], rate=0.5).step()
    values = torch.linalg.svdvals((before - p.detach()).double() / (0.5 * 1.5 ** 0.5))
    assert values.max() < 1.3 and values.min() > 0.5


def test_example_products_gradient_is_the_difference(example):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    tokens, up, offsets = new(30, 24), new(3, 24, 40), torch.tensor([0, 25, 25, 60], dtype=torch.int32, device="cuda")
    order = torch.randperm(60, generator=gen, device="cuda").int()
    position = torch.empty(60, dtype=torch.int32, device="cuda")
    position[order.long()] = torch.arange(60, dtype=torch.int32, device="cuda")
    dy = new(60, 40)

    def loss(tokens, up):
        rows = example.HandOut.apply(tokens, order, position.reshape(30, 2))
        return (example.Product.apply(rows, up, offsets).double() * dy.double()).sum()

    x, w = tokens.clone().requires_grad_(), up.clone().requires_grad_()
    loss(x, w).backward()
    wx, ww = new(30, 24), new(3, 24, 40)
    slope = float((x.grad.double() * wx).sum() + (w.grad.double() * ww).sum())
    # quadratic along the way: central differences are exact but for the rounding of 2,400 values of size 5 in f32
    with torch.no_grad():
        got = float(loss(tokens + 0.5 * wx, up + 0.5 * ww) - loss(tokens - 0.5 * wx, up - 0.5 * ww))
    assert abs(got - slope) <= 1e-5 * 2400 * 5 + 1e-5 * abs(slope)
    assert tb.tb_cuda_synchronize(torch.cuda.current_stream()) == 1
