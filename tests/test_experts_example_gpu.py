"""The example's wrappers of the experts' operators with tensors that lie in other ways than the C entry points take
them: the same results, or an error, and never another result without a word."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import experts_reference as ref  # noqa: E402
from tests.learner_reference import check  # noqa: E402
from tests.test_experts_gpu import KINDS, _gen, _normal, _whole  # noqa: E402
from tests.test_experts_path_gpu import example  # noqa: E402,F401

pytestmark = pytest.mark.gpu

OFFSETS = [0, 25, 25, 57]


def _lying(w, way):
    """The values of w [experts, in, out], lying another way."""
    e, n, m = w.shape
    if way == "transposed":
        return w.transpose(1, 2).contiguous().transpose(1, 2)
    if way == "slices":
        return torch.cat([w, w], 2)[..., :m]
    if way == "experts inside":
        return w.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    if way == "one for all":
        return w[:1].expand(e, n, m)
    return w


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("way", ("dense", "transposed", "slices", "experts inside", "one for all"))
def test_products_of_weights_that_lie_otherwise(example, way, kind):  # noqa: F811
    gen = _gen(41)
    rows, w = _normal(gen, 60, 24, kind=kind).requires_grad_(), _lying(_normal(gen, 3, 24, 40, kind=kind), way).requires_grad_()
    dy, off = _normal(gen, 60, 40, kind=kind), _whole(OFFSETS)
    y = example.Product.apply(rows, w, off)
    y.backward(dy)
    want, size = ref.product(rows.detach().double(), w.detach().double(), OFFSETS, False)
    (dx, dx_size), (dw, dw_size), depth = ref.product_backward(rows.detach().double(), w.detach().double(), OFFSETS, dy.double(), False)
    f32, used = kind == torch.float32, slice(0, 57)
    check("y", y.detach()[used], want[used], ref.sum_error(24, size[used], f32))
    check("dx", rows.grad[used], dx[used], ref.sum_error(40, dx_size[used], f32))
    check("dw", w.grad, dw, ref.sum_error(depth, dw_size, f32))
    assert w.grad.shape == w.shape


def test_products_of_what_does_not_go_together_are_refused(example):  # noqa: F811
    gen = _gen(42)
    rows, w, off = _normal(gen, 60, 24), _normal(gen, 3, 24, 40), _whole(OFFSETS)
    for bad in [(rows, w.bfloat16(), off), (rows.half(), w, off), (rows, w, off.long()), (rows, w, off[:-1]), (rows, w[:2], off),
                (rows[:, :23], w, off), (rows, w.transpose(1, 2), off), (rows, w, off.cpu()), (rows, w, off.repeat_interleave(2)[::2])]:
        with pytest.raises((TypeError, ValueError)):
            example.Product.apply(*bad)
    held, scale = example.quantised(w.transpose(1, 2))
    for bad in [(rows, held.short(), scale, off), (rows, held, scale.half(), off), (rows, held, scale[:, :-1], off),
                (rows, held.transpose(1, 2), scale, off), (rows, held, scale, off.long()), (rows[:, :23], held, scale, off)]:
        with pytest.raises((TypeError, ValueError)):
            example.product_8_bit(*bad)


def test_8_bit_products_of_weights_that_lie_otherwise(example):  # noqa: F811
    gen = _gen(43)
    rows, off = _normal(gen, 60, 24), _whole(OFFSETS)
    held, scale = example.quantised(_normal(gen, 3, 40, 24))
    want = example.product_8_bit(rows, held, scale, off)[:57]
    turned = held.transpose(1, 2).contiguous().transpose(1, 2), scale.T.contiguous().T
    assert torch.equal(example.product_8_bit(rows, *turned, off)[:57], want)
    wide = torch.cat([held, held], 2)[..., :24], torch.stack([scale, scale], 2)[..., 0]
    assert torch.equal(example.product_8_bit(rows, *wide, off)[:57], want)


@pytest.mark.parametrize("way", ("transposed", "slices", "experts inside"))
def test_momentum_of_parameters_that_lie_otherwise(example, way):  # noqa: F811
    """Two steps move the values as they move those of a dense parameter."""
    gen = _gen(44)
    values = _normal(gen, 2, 40, 60)
    plain, lying = torch.nn.Parameter(values.clone()), torch.nn.Parameter(_lying(values.clone(), way))
    moments = [example.OrthogonalMomentum([p], rate=0.5) for p in (plain, lying)]
    for _ in range(2):
        grad = _normal(gen, 2, 40, 60)
        plain.grad, lying.grad = grad.clone(), _lying(grad.clone(), way)
        for m in moments:
            m.step()
    assert torch.equal(plain.detach(), lying.detach()) and not torch.equal(plain.detach(), values)


def test_second_derivatives_are_refused(example):  # noqa: F811
    """The backward passes are kernels too, which autograd does not see into: an error, not a derivative without them."""
    gen = _gen(45)
    order = torch.randperm(60, generator=gen, device="cuda").int()
    position = torch.empty(60, dtype=torch.int32, device="cuda")
    position[order.long()] = torch.arange(60, dtype=torch.int32, device="cuda")
    position, off = position.reshape(30, 2), _whole([0, 25, 25, 60])
    x, w, logits, share = _normal(gen, 30, 24), _normal(gen, 3, 24, 40), _normal(gen, 30, 3), torch.rand((30, 2), generator=gen, device="cuda")
    gates, decay = _normal(gen, 2, 5, 72), _normal(gen, 24)
    reset, state = torch.zeros((2, 5), dtype=torch.uint8, device="cuda"), torch.zeros((2, 24), device="cuda")
    calls = [lambda v: example.HandOut.apply(v, order, position), lambda v: example.Product.apply(v.repeat(2, 1), w, off),
             lambda v: example.Combine.apply(v.repeat(2, 1), position, share),
             lambda v: example.RouteExperts.apply(logits + v[:, :3], torch.zeros(3, device="cuda"), 2)[0],
             lambda v: example.GatedRecurrence.apply(gates + v[:2, None, :1], decay, state, reset)[0],
             lambda v: example.GroupNormAct.apply(v.reshape(3, 10, 24), torch.ones(24, device="cuda"), torch.zeros(24, device="cuda"), 4)]
    for call in calls:
        v = x.clone().requires_grad_()
        (grad,) = torch.autograd.grad(call(v).square().sum(), v, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
            grad.square().sum().backward()
