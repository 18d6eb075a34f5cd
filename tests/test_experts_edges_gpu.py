"""The experts' operators on a B200 at the edges of their tiles, runs and numbers, against their 64-bit definitions."""
from __future__ import annotations

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

from tests import experts_reference as ref  # noqa: E402
from tests.learner_reference import check  # noqa: E402
from tests.test_experts_gpu import KINDS, _check_i8, _gen, _product_case, _synchronised, _whole  # noqa: E402

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


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("turned", (False, True), ids=("in_out", "out_in"))
def test_offsets_that_fall_stay_inside_the_tensors(kind, turned):
    """Runs that would overlap, where a tile's sums go through the workspace in parts: the sums of 16 tiles have room,
    and a run that begins again in front would have made 32 of them."""
    gen, rows, n, m, guard = _gen(31), 256, 2048, 128, 1 << 20
    desc, x, w, dy, _ = _product_case(gen, rows, [0] + [rows] * 8, n, m, kind, turned)
    need = tb.tb_cuda_experts_product_workspace(desc)
    for offsets in ([0, rows, 0, rows, 0, rows, 0, 0, rows], [0, rows] * 4 + [0], [rows, 0] * 4 + [rows], [9, 200, 3, 256, 100, 0, 7, 5, 250]):
        hold = torch.full((need + guard,), 171, dtype=torch.uint8, device="cuda")
        y, dx, dw = (torch.full((v.numel() + 4096,), 3.0, device="cuda").to(kind) for v in (dy, x, w))
        off = _whole(offsets)
        assert tb.tb_cuda_experts_product_device(desc, x, w, off, y, hold, torch.cuda.current_stream()) == 1
        assert tb.tb_cuda_experts_product_backward_device(desc, x, w, off, dy, dx, dw, hold, torch.cuda.current_stream()) == 1
        _synchronised()
        assert (hold[need:] == 171).all(), "written past the workspace"
        assert all((v[-4096:] == 3).all() for v in (y, dx, dw)), "written past an output"
        if offsets[1] == offsets[-1] == rows:  # a run begins where all in front of it end: the first has all rows
            want, size = ref.product(x.double(), w.double(), [0] + [rows] * 8, turned)
            check("y", y[:-4096].reshape(rows, m), want, ref.sum_error(n, size, kind == torch.float32))
