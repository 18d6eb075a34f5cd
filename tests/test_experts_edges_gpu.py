"""The experts' operators on a B200 at the edges of their tiles, runs and numbers, against their 64-bit definitions."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_experts_gpu import KINDS, _check_i8, _gen  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("last", (1, 16, 17, 33, 48, 80, 255))
def test_i8_last_tile_of_a_pair(last):
    """One dense layer, wide enough that two CTAs share a tile of 256 rows: a whole tile, then one of `last` rows.  The
    rows behind them are of no expert, and hold what no row may show."""
    gen = _gen(last)
    n, m, rows = 400, 4096, 256 + last
    q = torch.randint(-127, 128, (rows + 40, n), generator=gen, device="cuda").to(torch.int8)
    q[rows:] = -128
    w = torch.randint(-127, 128, (1, m, n), generator=gen, device="cuda").to(torch.int8)
    _check_i8(q, torch.rand(rows + 40, generator=gen, device="cuda"), w, torch.rand((1, m), generator=gen, device="cuda"), [0, rows],
              KINDS[last % 3])
