"""The experts' operators on a B200 at the edges of their tiles, runs and numbers, against their 64-bit definitions."""
from __future__ import annotations

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

from tests import experts_reference as ref  # noqa: E402
from tests.learner_reference import check  # noqa: E402
from tests.test_experts_gpu import KINDS, _check_i8, _check_product, _gen, _normal, _product_case, _synchronised, _whole, _work  # noqa: E402

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


FEW = [  # rows, offsets, in, out: runs that begin and end inside four rows, rows of no expert among them
    (11, [1, 2, 4, 4, 9, 10], 70, 130),
    (7, [0, 1, 3, 6], 64, 96),
    (8, [2, 2, 3, 7, 7, 7], 33, 40),
    (16, [0, 0, 5, 6, 16], 520, 520),
]


@pytest.mark.parametrize("turned", (False, True), ids=("in_out", "out_in"))
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", FEW, ids=str)
def test_few_rows_of_several_experts(shape, kind, turned):
    rows, offsets, n, m = shape
    _check_product(_gen(rows + n), rows, offsets, n, m, kind, turned)


@pytest.mark.parametrize("shape", FEW, ids=str)
def test_few_8_bit_rows_of_several_experts(shape):
    rows, offsets, n, m = shape
    gen, e = _gen(rows), len(offsets) - 1
    q = torch.randint(-128, 128, (rows, n), generator=gen, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (e, m, n), generator=gen, device="cuda").to(torch.int8)
    _check_i8(q, torch.rand(rows, generator=gen, device="cuda"), w, torch.rand((e, m), generator=gen, device="cuda"), offsets, KINDS[rows % 3])


def test_products_over_2_31_elements_with_the_room_they_ask_for():
    """Each call has the workspace that its own query names; the last expert's rows lie far behind 2^31 elements."""
    rows, n, m, tail = 4_300_000, 512, 520, 700
    gen = _gen(16)
    x, dy = (torch.empty((rows, width), dtype=torch.bfloat16, device="cuda") for width in (n, m))
    for v in (x, dy):
        for part in v.split(1 << 19):
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda"))
    w = _normal(gen, 2, m, n, kind=torch.bfloat16, scale=0.05)
    got = []
    for xs, dys, offsets in [(x, dy, [0, rows - tail, rows]), (x[-tail:].clone(), dy[-tail:].clone(), [0, 0, tail])]:
        count = xs.shape[0]
        desc = tb.ExpertProductDesc(rows=count, experts=2, in_width=n, out_width=m, weight_order=tb.TB_WEIGHT_OUT_IN, type=tb.TB_TYPE_BF16)
        work, off = torch.empty(tb.tb_cuda_experts_product_workspace(desc), dtype=torch.uint8, device="cuda"), _whole(offsets)
        y, dx, dw = torch.empty_like(dys), torch.empty_like(xs), torch.empty_like(w)
        assert tb.tb_cuda_experts_product_device(desc, xs, w, off, y, work, torch.cuda.current_stream()) == 1
        assert tb.tb_cuda_experts_product_backward_device(desc, xs, w, off, dys, dx, dw, work, torch.cuda.current_stream()) == 1
        _synchronised()
        got.append((y[-tail:].clone(), dx[-tail:].clone(), dw[1]))
        del work, y, dx
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    right, left = x[-tail:].double(), dy[-tail:].double().T
    want, size = left @ right, left.abs() @ right.abs()
    for _, _, dw in got:  # the sums' parts go by the average run, so that the bits may differ
        check("dw", dw, want, ref.sum_error(tail, size))
    del x, dy
    torch.cuda.empty_cache()
