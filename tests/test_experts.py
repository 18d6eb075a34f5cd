"""The experts' operators without a GPU: what the entry points refuse before they touch a device, and the 64-bit
definitions' gradients against differences."""
from __future__ import annotations

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

from tests import experts_reference as ref  # noqa: E402

FAKE = 1 << 20  # an aligned address that nothing reads: every call below is refused


def _product(**change):
    return tb.ExpertProductDesc(**{**dict(rows=8, experts=2, in_width=16, out_width=24, type=1), **change})


@pytest.mark.parametrize("change", [
    dict(rows=0), dict(experts=0), dict(in_width=0), dict(out_width=0), dict(type=3), dict(type=-1), dict(weight_order=2),
    dict(experts=1025), dict(rows=2 ** 31 - 255), dict(in_width=2 ** 31 - 255), dict(out_width=2 ** 31), dict(in_stride=15),
    dict(din_stride=15), dict(out_stride=23), dict(weight_row_stride=23), dict(weight_order=1, weight_row_stride=15),
    dict(weight_expert_stride=16 * 24 - 1), dict(in_stride=2 ** 61), dict(weight_row_stride=2 ** 61),
    dict(weight_expert_stride=2 ** 60), dict(rows=2 ** 31 - 300, out_width=2 ** 31 - 300)], ids=str)
def test_product_refuses_descriptors(change):
    d = _product(**change)
    assert tb.tb_cuda_experts_product_workspace(d) == 0
    assert tb.tb_cuda_experts_product_device(d, FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE) == 0
    assert tb.tb_cuda_experts_product_backward_device(d, FAKE, FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE) == 0


def test_product_refuses_pointers():
    assert tb.tb_cuda_experts_product_workspace(_product()) > 0
    # x weight offsets y workspace
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (4, None), (0, FAKE + 1), (1, FAKE + 1), (2, FAKE + 2),
                   (3, 2 * FAKE + 1), (4, 3 * FAKE + 8), (3, FAKE), (4, FAKE), (4, 2 * FAKE)]:
        args = [FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_experts_product_device(_product(), *args) == 0, (i, bad)
    # x weight offsets dy dx dweight workspace
    good = [FAKE, FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE]
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (6, None), (0, FAKE + 1), (1, FAKE + 1), (2, FAKE + 2),
                   (3, FAKE + 1), (4, FAKE + 1), (5, FAKE + 1), (6, FAKE + 8), (4, FAKE), (5, FAKE), (5, 2 * FAKE), (6, FAKE)]:
        args = list(good)
        args[i] = bad
        assert tb.tb_cuda_experts_product_backward_device(_product(), *args) == 0, (i, bad)
    assert tb.tb_cuda_experts_product_backward_device(_product(), *good[:4], None, None, 4 * FAKE) == 0
    assert tb.load_library().tb_cuda_experts_product_device(None, FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE, None) == 0


@pytest.mark.parametrize("change", [dict(rows=0), dict(width=0), dict(type=3), dict(rows=2 ** 31), dict(x_stride=15), dict(q_stride=15),
                                    dict(x_stride=2 ** 61), dict(q_stride=2 ** 62)], ids=str)
def test_quantise_refuses_descriptors(change):
    d = tb.QuantiseDesc(**{**dict(rows=8, width=16, type=1), **change})
    assert tb.tb_cuda_quantise_rows_device(d, FAKE, 2 * FAKE, 3 * FAKE) == 0


def test_quantise_refuses_pointers():
    for i, bad in [(0, None), (1, None), (2, None), (0, FAKE + 1), (2, FAKE + 2), (1, FAKE), (2, FAKE), (2, 2 * FAKE)]:
        args = [FAKE, 2 * FAKE, 3 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_quantise_rows_device(tb.QuantiseDesc(rows=8, width=16, type=1), *args) == 0, (i, bad)


def _i8(**change):
    return tb.ExpertProductI8Desc(**{**dict(rows=8, experts=2, in_width=16, out_width=24, type=1), **change})


@pytest.mark.parametrize("change", [
    dict(rows=0), dict(experts=0), dict(in_width=0), dict(out_width=0), dict(type=3), dict(experts=1025), dict(rows=2 ** 31 - 255),
    dict(in_width=131072), dict(out_width=2 ** 31), dict(in_stride=15), dict(out_stride=23), dict(weight_row_stride=15),
    dict(weight_expert_stride=16 * 24 - 1), dict(in_stride=2 ** 61)], ids=str)
def test_i8_refuses_descriptors(change):
    d = _i8(**change)
    assert tb.tb_cuda_experts_product_i8_workspace(d) == 0
    assert tb.tb_cuda_experts_product_i8_device(d, *[FAKE] * 5, 2 * FAKE, 3 * FAKE) == 0


def test_i8_refuses_pointers():
    assert tb.tb_cuda_experts_product_i8_workspace(_i8()) > 0
    # q q_scale weight weight_scale offsets y workspace
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (6, None), (1, FAKE + 2), (3, FAKE + 2),
                   (4, FAKE + 2), (5, FAKE + 1), (6, FAKE + 8), (5, FAKE), (6, FAKE), (6, 2 * FAKE)]:
        args = [FAKE] * 5 + [2 * FAKE, 3 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_experts_product_i8_device(_i8(), *args) == 0, (i, bad)


def _orthogonal(**change):
    return tb.OrthogonaliseDesc(**{**dict(matrices=2, rows=8, columns=12, type=0, steps=5, a=3.4445, b=-4.775, c=2.0315, epsilon=1e-7,
                                          scale=1.0), **change})


@pytest.mark.parametrize("change", [
    dict(matrices=0), dict(rows=0), dict(columns=0), dict(type=3), dict(steps=0), dict(steps=65), dict(rows=65537), dict(columns=65537),
    dict(matrices=65536), dict(epsilon=-1e-9), dict(epsilon=float("nan")), dict(in_row_stride=11), dict(out_row_stride=11),
    dict(in_matrix_stride=95), dict(out_matrix_stride=95), dict(in_row_stride=2 ** 61), dict(out_matrix_stride=2 ** 61)], ids=str)
def test_orthogonalise_refuses_descriptors(change):
    d = _orthogonal(**change)
    assert tb.tb_cuda_orthogonalise_workspace(d) == 0
    assert tb.tb_cuda_orthogonalise_device(d, FAKE, 2 * FAKE, 3 * FAKE) == 0


def test_orthogonalise_refuses_pointers():
    assert tb.tb_cuda_orthogonalise_workspace(_orthogonal()) > 0
    for i, bad in [(0, None), (1, None), (2, None), (0, FAKE + 2), (1, FAKE + 2), (2, FAKE + 8), (2, FAKE), (2, 2 * FAKE)]:
        args = [FAKE, 2 * FAKE, 3 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_orthogonalise_device(_orthogonal(), *args) == 0, (i, bad)
    assert tb.tb_cuda_orthogonalise_device(_orthogonal(out_row_stride=16), FAKE, FAKE, 3 * FAKE) == 0  # in place: the same strides


def _combine(**change):
    return tb.ExpertCombineDesc(**{**dict(tokens=4, rows=8, width=16, top_k=2, type=1), **change})


@pytest.mark.parametrize("change", [
    dict(tokens=0), dict(rows=0), dict(width=0), dict(top_k=0), dict(top_k=33), dict(type=3), dict(rows_stride=15), dict(out_stride=15),
    dict(tokens=2 ** 31), dict(rows=2 ** 31), dict(width=2 ** 60)], ids=str)
def test_hand_out_refuses_descriptors(change):
    d = _combine(**change)
    assert tb.tb_cuda_hand_out_experts_device(d, FAKE, FAKE, FAKE, 2 * FAKE) == 0
    assert tb.tb_cuda_hand_out_experts_backward_device(d, FAKE, FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE) == 0


def test_hand_out_refuses_pointers():
    for i, bad in [(0, None), (1, None), (3, None), (3, FAKE), (0, FAKE + 1), (1, FAKE + 2), (2, FAKE + 2), (3, FAKE + 1)]:
        args = [FAKE, FAKE, FAKE, 2 * FAKE]
        args[i] = bad
        assert tb.tb_cuda_hand_out_experts_device(_combine(), *args) == 0, (i, bad)
    good = [FAKE, FAKE, FAKE, FAKE, 2 * FAKE, 3 * FAKE]  # x position weights drows dx dweights
    for i, bad in [(0, None), (1, None), (3, None), (4, FAKE), (5, FAKE), (5, 2 * FAKE), (0, FAKE + 1), (1, FAKE + 2), (2, FAKE + 2),
                   (3, FAKE + 1), (4, 2 * FAKE + 1), (5, 3 * FAKE + 2)]:
        args = list(good)
        args[i] = bad
        assert tb.tb_cuda_hand_out_experts_backward_device(_combine(), *args) == 0, (i, bad)
    assert tb.tb_cuda_hand_out_experts_backward_device(_combine(), *good[:4], None, None) == 0


@pytest.mark.parametrize("turned", (False, True))
def test_product_gradient_is_the_difference(turned):
    gen = torch.Generator().manual_seed(1)
    f64 = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    offsets, x, dy = [1, 4, 4, 9], f64(10, 5), f64(10, 7)
    w = f64(3, 7, 5) if turned else f64(3, 5, 7)
    (dx, _), (dw, _), _ = ref.product_backward(x, w, offsets, dy, turned)
    loss = lambda x, w: (ref.product(x, w, offsets, turned)[0] * dy)[1:9].sum()  # noqa: E731
    wx, ww, h = f64(10, 5), f64(*w.shape), 1e-6
    assert torch.allclose((dx * wx)[1:9].sum(), (loss(x + h * wx, w) - loss(x - h * wx, w)) / (2 * h), rtol=1e-6)
    assert torch.allclose((dw * ww).sum(), (loss(x, w + h * ww) - loss(x, w - h * ww)) / (2 * h), rtol=1e-6)
    assert (dw[1] == 0).all()


def test_orthogonalised_update_has_singular_values_near_one():
    gen = torch.Generator().manual_seed(2)
    g = torch.randn((2, 30, 50), generator=gen, dtype=torch.float64)
    out = ref.orthogonalise(g, 5, 3.4445, -4.7750, 2.0315, 1e-7, 1.0)
    values = torch.linalg.svdvals(out)
    assert values.max() < 1.3 and values.min() > 0.6
    assert torch.allclose(out, ref.orthogonalise(g.transpose(1, 2), 5, 3.4445, -4.7750, 2.0315, 1e-7, 1.0).transpose(1, 2))
