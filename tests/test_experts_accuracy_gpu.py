"""The digits of the experts' operators' f32 results on a B200: products of planes and updates in pairs keep what
tests/experts_accuracy.py says that their arithmetic keeps, small values beside large ones among them."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import experts_accuracy as exact  # noqa: E402
from tests import experts_reference as ref  # noqa: E402
from tests.test_experts_gpu import QUINTIC, _gen, _normal, _orthogonalise  # noqa: E402

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
