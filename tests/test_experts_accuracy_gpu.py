"""The digits of the experts' operators' f32 results on a B200: products of planes and updates in pairs keep what
tests/experts_accuracy.py says that their arithmetic keeps, small values beside large ones among them."""
from __future__ import annotations

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

from tests import experts_accuracy as exact  # noqa: E402
from tests import experts_reference as ref  # noqa: E402
from tests.test_experts_gpu import QUINTIC, _gen, _normal, _orthogonalise, _product_case, _synchronised, _whole, _work  # noqa: E402

pytestmark = pytest.mark.gpu


def _update(g, epsilon=0.0):
    out = torch.empty_like(g)
    _orthogonalise(g, out, epsilon=epsilon)
    return out.double(), ref.orthogonalise(g, 5, *QUINTIC.values(), epsilon, 1.0)


@pytest.mark.parametrize("shape", [(8, 128, 256), (2, 33, 20), (1, 600, 700), (1, 40, 3000), (1, 1500, 90), (1, 1300, 1100)], ids=str)
def test_update_is_as_good_as_f32(shape):
    """Two bits more than plain f32 arithmetic on the same gradient at most, and no more than the kernel's rule allows."""
    g = _normal(_gen(sum(shape)), *shape)
    got, want = _update(g)
    plain = exact.rms(exact.update_in_f32(g, 5, *QUINTIC.values(), 0.0, 1.0) - want)
    rule = exact.rms(exact.update_with_errors(g, 5, *QUINTIC.values(), 0.0, 1.0) - want)
    assert exact.rms(got - want) <= min(4 * plain, rule)


@pytest.mark.parametrize("shape", [(1, 256, 512), (2, 512, 256), (1, 40, 3000), (1, 90, 60)], ids=str)
@pytest.mark.parametrize("factor", (1e-3, 1e-5, 1e-6))
def test_update_of_rows_far_smaller_than_others(shape, factor):
    """Every other row (column of a matrix taller than wide) a small factor of the rest: it keeps its own digits."""
    g = _normal(_gen(sum(shape)), *shape)
    tall = shape[1] > shape[2]
    (g.transpose(1, 2) if tall else g)[:, ::2] *= factor
    got, want = _update(g)
    rule = exact.update_with_errors(g, 5, *QUINTIC.values(), 0.0, 1.0)
    if tall:
        got, want, rule = (v.transpose(1, 2) for v in (got, want, rule))
    for rows in (slice(0, None, 2), slice(1, None, 2)):
        assert exact.rms((got - want)[:, rows]) <= exact.rms((rule - want)[:, rows])


def _products(rows, offsets, n, m, turned, x_scale=1.0, w_scale=1.0):
    """y, dx and dw of f32 tensors, each with its definition and the size of its sums."""
    desc, x, w, dy, used = _product_case(_gen(rows + n), rows, offsets, n, m, torch.float32, turned)
    x *= x_scale
    w *= w_scale
    work, off = _work(tb.tb_cuda_experts_product_workspace(desc)), _whole(offsets)
    y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w)
    assert tb.tb_cuda_experts_product_device(desc, x, w, off, y, work, torch.cuda.current_stream()) == 1
    assert tb.tb_cuda_experts_product_backward_device(desc, x, w, off, dy, dx, dw, work, torch.cuda.current_stream()) == 1
    _synchronised()
    x, w, dy = x.double(), w.double(), dy.double()
    out = []
    for e, r in ref.runs(offsets, rows):
        m_e = w[e].T if turned else w[e]
        left, right = (dy[r], x[r]) if turned else (x[r], dy[r])
        out += [("y", n, y[r], x[r] @ m_e, exact.size(x[r], m_e)), ("dx", m, dx[r], dy[r] @ m_e.T, exact.size(dy[r], m_e.T)),
                ("dw", r.stop - r.start, dw[e], left.T @ right, exact.size(left.T, right))]
    return out


SUMS = [(64, [0, 64], 64, 64), (512, [0, 512], 512, 512), (600, [0, 89, 600], 512, 4096), (4500, [0, 4096, 4500], 4096, 64)]


@pytest.mark.parametrize("turned", (False, True), ids=("in_out", "out_in"))
@pytest.mark.parametrize("shape", SUMS, ids=str)
def test_f32_products_keep_their_digits(shape, turned):
    """With the smallest products of planes left out the root mean square is 2.4e-6 to 4.5e-6, with one sum over all of
    4,096 in the tensor cores 4e-6; the rule allows 7.8e-7 to 9.6e-7."""
    for name, depth, got, want, size in _products(*shape, turned):
        assert exact.rms((got - want) / size) <= exact.sum_error(depth), (name, depth)


@pytest.mark.parametrize("exponents", [(-118, 20), (-124, 24), (30, -120), (-126, 120), (100, 20)], ids=str)
def test_f32_products_of_small_and_large_values(exponents):
    """Down to f32's least normal numbers: a value is held to 2^-148 at least, and the other factor is as exact as ever."""
    a, b = (2.0 ** e for e in exponents)
    for name, depth, got, want, size in _products(300, [0, 120, 300], 512, 160, False, a, b):
        if name == "y":
            least = 2.0 ** -148 * depth ** 0.5 * (a + b * 512 ** -0.5)
            assert exact.rms((got - want) / size) <= exact.sum_error(depth) + least / float(size.min()), name
        elif name == "dx" if b < 1 else name == "dw":
            least = 2.0 ** -148 * depth ** 0.5
            assert exact.rms((got - want) / size) <= exact.sum_error(depth) + least / float(size.min()), name


def test_f32_products_of_the_largest_values():
    """Times one: nothing on the way passes f32's range, and each comes back as it was."""
    top = torch.finfo(torch.float32).max
    x = torch.tensor([top, -top, 0.9999 * top, 2.0 ** 127, 1.0, 3.0e38], device="cuda").repeat(11)[:64].repeat(64, 1).contiguous()
    desc = tb.ExpertProductDesc(rows=64, experts=1, in_width=64, out_width=64, weight_order=tb.TB_WEIGHT_OUT_IN, type=tb.TB_TYPE_F32)
    y = torch.empty_like(x)
    assert tb.tb_cuda_experts_product_device(desc, x, torch.eye(64, device="cuda"), None, y, _work(tb.tb_cuda_experts_product_workspace(desc))) == 1
    torch.cuda.synchronize()
    assert torch.equal(y, x)
