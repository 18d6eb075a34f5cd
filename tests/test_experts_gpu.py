"""The experts' operators on a B200 against their 64-bit definitions: handing out, products and both gradients, 8-bit
products, orthogonalised updates, at the sizes, orders and contents where they can go wrong."""
from __future__ import annotations

import pytest

import turbinator_c_b200 as tb

torch = pytest.importorskip("torch")

from tests import experts_reference as ref  # noqa: E402
from tests.learner_reference import U, check  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {torch.float32: tb.TB_TYPE_F32, torch.bfloat16: tb.TB_TYPE_BF16, torch.float16: tb.TB_TYPE_F16}
KINDS = list(TYPES)
NAN = float("nan")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(gen, *shape, kind=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(kind)


def _whole(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _work(need):
    assert need > 0
    return torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # NaN in every type: scratch is not read as it was


def _inside(shape, kind, pad, shift=0):
    """A tensor of `shape` whose rows lie `pad` elements apart and start `shift` elements into their storage, NaN around
    them."""
    rows = 1
    for n in shape[:-1]:
        rows *= n
    flat = torch.full((rows * (shape[-1] + pad) + shift,), NAN, device="cuda").to(kind)
    strides, step = [1], shape[-1] + pad
    for n in reversed(shape[:-1]):
        strides.insert(0, step)
        step *= n
    return flat.as_strided(shape, strides, shift)


def _synchronised():
    assert tb.tb_cuda_synchronize(torch.cuda.current_stream()) == 1


# ---- products ----

def _product_case(gen, rows, offsets, n, m, kind, turned, pads=(0, 0, 0, 0), shift=0):
    e = len(offsets) - 1
    x, dy = _inside((rows, n), kind, pads[0], shift), _inside((rows, m), kind, pads[1], shift)
    w = _inside((e, m, n) if turned else (e, n, m), kind, pads[2], shift)
    x.copy_(_normal(gen, rows, n)), dy.copy_(_normal(gen, rows, m)), w.copy_(_normal(gen, *w.shape, scale=n ** -0.5))
    desc = tb.ExpertProductDesc(rows=rows, experts=e, in_width=n, out_width=m, in_stride=n + pads[0], din_stride=n + pads[3],
                                out_stride=m + pads[1], weight_row_stride=w.stride(1), weight_expert_stride=w.stride(0),
                                weight_order=tb.TB_WEIGHT_OUT_IN if turned else tb.TB_WEIGHT_IN_OUT, type=TYPES[kind])
    used = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for _, r in ref.runs(offsets, rows):
        used[r] = True
    x[~used], dy[~used] = NAN, NAN  # rows of no expert are not used
    return desc, x, w, dy, used


def _check_product(gen, rows, offsets, n, m, kind, turned, pads=(0, 0, 0, 0), shift=0, given=True):
    desc, x, w, dy, used = _product_case(gen, rows, offsets, n, m, kind, turned, pads, shift)
    off = _whole(offsets) if given else None
    work = _work(tb.tb_cuda_experts_product_workspace(desc))
    y, dx, dw = _inside((rows, m), kind, pads[1], shift), _inside((rows, n), kind, pads[3], shift), _inside(tuple(w.shape), kind, pads[2], shift)
    y.fill_(3.0), dx.fill_(5.0)
    assert tb.tb_cuda_experts_product_device(desc, x, w, off, y, work, torch.cuda.current_stream()) == 1
    assert tb.tb_cuda_experts_product_backward_device(desc, x, w, off, dy, dx, dw, work, torch.cuda.current_stream()) == 1
    _synchronised()
    f32 = kind == torch.float32
    want, size = ref.product(x.double(), w.double(), offsets, turned)
    check("y", y[used], want[used], ref.sum_error(n, size[used], f32))
    (dx_want, dx_size), (dw_want, dw_size), depth = ref.product_backward(x.double(), w.double(), offsets, dy.double(), turned)
    check("dx", dx[used], dx_want[used], ref.sum_error(m, dx_size[used], f32))
    check("dw", dw, dw_want, ref.sum_error(depth, dw_size, f32))
    assert (y[~used] == 3).all() and (dx[~used] == 5).all(), "rows of no expert were written"
    return desc, x, w, dy, off, y, dx, dw, work


SHAPES = [  # rows, offsets, in, out
    (1, [0, 1], 8, 8),
    (1, [0, 1], 300, 70),
    (5, [0, 0, 5, 5], 64, 128),
    (40, [0, 0, 0, 0], 32, 24),
    (77, [3, 3, 20, 21, 70], 72, 200),
    (129, [0, 64, 129], 129, 257),
    (300, [0, 1, 2, 3, 290], 256, 384),
    (700, [0, 250, 512, 700], 513, 320),
    (1500, [0, 3, 1499], 40, 1025),
]


@pytest.mark.parametrize("turned", (False, True), ids=("in_out", "out_in"))
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product_and_gradients(shape, kind, turned):
    rows, offsets, n, m = shape
    _check_product(_gen(rows + n), rows, offsets, n, m, kind, turned)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("pads,shift", [((8, 16, 8, 0), 0), ((3, 1, 5, 7), 0), ((0, 0, 0, 0), 1), ((1, 0, 0, 9), 3)], ids=str)
def test_product_strides_and_alignment(kind, pads, shift):
    _check_product(_gen(5), 211, [0, 80, 211], 96, 136, kind, False, pads, shift)
    _check_product(_gen(6), 90, [2, 40, 41, 88], 56, 72, kind, True, pads, shift)


@pytest.mark.parametrize("kind", (torch.bfloat16, torch.float32), ids=str)
def test_product_of_one_expert_without_offsets(kind):
    for rows in (1, 33, 400):
        _check_product(_gen(rows), rows, [0, rows], 136, 264, kind, True, given=False)


@pytest.mark.parametrize("kind", (torch.bfloat16, torch.float32), ids=str)
@pytest.mark.parametrize("count", (2, 150))
def test_product_of_many_rows_and_ragged_runs(kind, count):
    gen = _gen(count)
    edges = torch.randint(0, 9001, (count - 1,), generator=gen, device="cuda").sort().values.tolist()
    _check_product(gen, 9000, [0, *edges, 9000], 200, 260, kind, count == 2)


@pytest.mark.parametrize("kind", (torch.bfloat16, torch.float32), ids=str)
def test_product_sums_a_long_axis(kind):
    """Few and narrow tiles, much to sum in each: the inputs' width, the rows of one expert."""
    _check_product(_gen(1), 24, [0, 11, 24], 4096, 96, kind, True)
    _check_product(_gen(2), 20011, [0, 20011], 64, 72, kind, False)


@pytest.mark.parametrize("kind", (torch.bfloat16, torch.float16), ids=str)
@pytest.mark.parametrize("turned", (False, True), ids=("in_out", "out_in"))
def test_product_of_many_wide_tiles(kind, turned):
    """Runs that end anywhere in a tile of 256 x 256, and widths past its edges."""
    _check_product(_gen(3), 20003, [0, 9000, 9001, 19700], 200, 1100, kind, turned)
    _check_product(_gen(4), 5000, [3, 2100, 2100, 4990], 1100, 1304, kind, turned)


def test_product_offsets_out_of_range_are_taken_into_it():
    gen = _gen(8)
    desc, x, w, dy, _ = _product_case(gen, 60, [0, 20, 40, 60], 64, 64, torch.bfloat16, False)
    work, y, dw = _work(tb.tb_cuda_experts_product_workspace(desc)), torch.full((60, 64), 3.0, device="cuda").bfloat16(), torch.empty_like(w)
    off = [-7, 25, 40, 2 ** 31 - 1]
    assert tb.tb_cuda_experts_product_device(desc, x, w, _whole(off), y, work) == 1
    assert tb.tb_cuda_experts_product_backward_device(desc, x, w, _whole(off), dy, None, dw, work) == 1
    torch.cuda.synchronize()
    want, size = ref.product(x.double(), w.double(), [0, 25, 40, 60], False)
    check("y", y, want, ref.sum_error(64, size))
    _, (dw_want, dw_size), depth = ref.product_backward(x.double(), w.double(), [0, 25, 40, 60], dy.double(), False)
    check("dw", dw, dw_want, ref.sum_error(depth, dw_size))


def test_product_keeps_what_is_not_finite_to_its_row_and_channel():
    gen = _gen(9)
    for kind in KINDS:
        desc, x, w, dy, _ = _product_case(gen, 300, [0, 130, 290], 192, 160, kind, False)
        x[7], dy[131, 3], w[1, 5, 9] = NAN, float("inf"), NAN
        work = _work(tb.tb_cuda_experts_product_workspace(desc))
        y, dx, dw = torch.empty((300, 160), device="cuda").to(kind), torch.empty((300, 192), device="cuda").to(kind), torch.empty_like(w)
        off = _whole([0, 130, 290])
        assert tb.tb_cuda_experts_product_device(desc, x, w, off, y, work) == 1
        assert tb.tb_cuda_experts_product_backward_device(desc, x, w, off, dy, dx, dw, work) == 1
        torch.cuda.synchronize()
        bad = ~torch.isfinite(y[:290])
        assert bad[7].all() and bad[130:, 9].all() and int(bad.sum()) == 160 + 160
        bad = ~torch.isfinite(dx[:290])
        assert bad[131].all() and bad[130:, 5].all() and int(bad.sum()) == 192 + 159
        bad = ~torch.isfinite(dw)
        assert bad[0].all() and bad[1, :, 3].all() and int(bad.sum()) == 192 * 160 + 192


@pytest.mark.parametrize("kind", (torch.bfloat16, torch.float32), ids=str)
def test_product_gives_the_same_bits_and_halves_alone(kind):
    gen = _gen(10)
    desc, x, w, dy, off, y, dx, dw, work = _check_product(gen, 1000, [0, 300, 950], 320, 512, kind, False)
    for _ in range(3):
        again = [torch.full_like(v, 1.0) for v in (y, dx, dw)]
        assert tb.tb_cuda_experts_product_device(desc, x, w, off, again[0], work) == 1
        assert tb.tb_cuda_experts_product_backward_device(desc, None, w, off, dy, again[1], None, work) == 1
        assert tb.tb_cuda_experts_product_backward_device(desc, x, None, off, dy, None, again[2], work) == 1
        torch.cuda.synchronize()
        assert torch.equal(again[0][:950], y[:950]) and torch.equal(again[1][:950], dx[:950]) and torch.equal(again[2], dw)


def test_product_gradient_is_the_difference():
    gen = _gen(11)
    rows, offsets, n, m = 90, [0, 33, 90], 40, 56
    desc, x, w, dy, _ = _product_case(gen, rows, offsets, n, m, torch.float32, False)
    work, off = _work(tb.tb_cuda_experts_product_workspace(desc)), _whole(offsets)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    assert tb.tb_cuda_experts_product_backward_device(desc, x, w, off, dy, dx, dw, work) == 1
    wx, ww = _normal(gen, rows, n), _normal(gen, *w.shape)

    def loss(t):
        y = torch.empty((rows, m), device="cuda")
        assert tb.tb_cuda_experts_product_device(desc, x + t * wx, w + t * ww, off, y, work) == 1
        return float((y.double() * dy.double()).sum())

    # the loss is a quadratic in t: central differences are exact but for its values' rounding
    size = float((x.abs().double() @ w.abs().double().sum(0)).mean()) * rows * m ** 0.5
    slope = float((dx.double() * wx).sum() + (dw.double() * ww).sum())
    assert abs((loss(0.5) - loss(-0.5)) - slope) <= 1e-5 * (abs(slope) + size)


# ---- 8-bit products ----

@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,width,pad", [(1, 1, 0), (3, 7, 0), (5, 4096, 0), (64, 129, 3), (200, 1000, 8), (2, 20000, 0),
                                            (2051, 33, 0), (3001, 512, 8), (2100, 4100, 0)])
def test_quantise_is_its_definition(kind, rows, width, pad):
    x = _inside((rows, width), kind, pad, pad % 2)
    x.copy_(_normal(_gen(rows), rows, width, scale=3.0) * torch.logspace(-3, 3, rows, device="cuda")[:, None])
    q, scale = torch.full((rows, width + pad), 99, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    desc = tb.QuantiseDesc(rows=rows, width=width, x_stride=width + pad, q_stride=width + pad, type=TYPES[kind])
    assert tb.tb_cuda_quantise_rows_device(desc, x, q, scale) == 1
    torch.cuda.synchronize()
    want, want_scale = ref.quantise(x.cpu())
    assert torch.equal(q[:, :width].cpu(), want) and torch.equal(scale.cpu(), want_scale)
    assert (q[:, width:] == 99).all()


def test_quantise_corners():
    x = torch.zeros((9, 24), device="cuda")
    x[1, 3], x[2, 4], x[3, 5] = NAN, float("inf"), -float("inf")
    x[4], x[5, 2], x[6, 1], x[7, 0] = 1e-40, 2.0 ** -121, 3.4e38, -5.0
    x[8] = torch.arange(24, device="cuda") - 11.5  # ties at whole numbers and a half
    x[8, 0] = 127.0
    q, scale = torch.empty((9, 24), dtype=torch.int8, device="cuda"), torch.empty(9, device="cuda")
    assert tb.tb_cuda_quantise_rows_device(tb.QuantiseDesc(rows=9, width=24, type=0), x, q, scale) == 1
    torch.cuda.synchronize()
    want, want_scale = ref.quantise(x.cpu())
    assert torch.equal(q.cpu(), want)
    assert torch.equal(torch.isnan(scale.cpu()), torch.isnan(want_scale)) and torch.equal(scale.cpu().nan_to_num(-1), want_scale.nan_to_num(-1))
    assert torch.isnan(scale[1:4]).all() and scale[0] == 0 and scale[4] == 0 and q[7, 0] == -127


def _check_i8(q, q_scale, w, w_scale, offsets, kind, given=True):
    rows, n = q.shape
    e, m = w_scale.shape
    desc = tb.ExpertProductI8Desc(rows=rows, experts=e, in_width=n, out_width=m, in_stride=q.stride(0) if rows > 1 else 0,
                                  weight_expert_stride=w.stride(0) if e > 1 else 0, weight_row_stride=w.stride(1) if m > 1 else 0,
                                  type=TYPES[kind])
    work, y = _work(tb.tb_cuda_experts_product_i8_workspace(desc)), torch.full((rows, m), 3.0, device="cuda").to(kind)
    assert tb.tb_cuda_experts_product_i8_device(desc, q, q_scale, w, w_scale, _whole(offsets) if given else None, y, work,
                                                torch.cuda.current_stream()) == 1
    _synchronised()
    used = torch.zeros(rows, dtype=torch.bool, device="cuda")
    want = torch.zeros((rows, m), dtype=torch.float64, device="cuda")
    for k, r in ref.runs(offsets, rows):
        used[r] = True
        want[r] = (q[r].double() @ w[k].double().T) * (q_scale[r, None].double() * w_scale[k].double())
    # the sum is exact; its conversion to f32 and two products are one U each; f16 has infinities from 65,520 on
    error, past = 4 * U * want[used].abs(), torch.isinf(want.to(kind))
    check("y", y[used], torch.where(past, want.sign() * float("inf"), want)[used], error)
    assert (y[~used] == 3).all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", SHAPES + [(9, [0, 9], 16, 4000), (2, [0, 1, 2], 33, 5)], ids=str)
def test_i8_product(shape, kind):
    rows, offsets, n, m = shape
    gen, e = _gen(rows + m), len(offsets) - 1
    q = torch.randint(-128, 128, (rows, n), generator=gen, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (e, m, n), generator=gen, device="cuda").to(torch.int8)
    _check_i8(q, torch.rand(rows, generator=gen, device="cuda"), w, torch.rand((e, m), generator=gen, device="cuda"), offsets, kind)


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_i8_product_of_many_wide_tiles(kind):
    gen = _gen(21)
    q = torch.randint(-128, 128, (20003, 300), generator=gen, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (3, 1100, 300), generator=gen, device="cuda").to(torch.int8)
    _check_i8(q, torch.rand(20003, generator=gen, device="cuda"), w, torch.rand((3, 1100), generator=gen, device="cuda"), [0, 9000, 9001, 19700], kind)


@pytest.mark.parametrize("pad,shift", [(16, 0), (5, 0), (0, 1), (3, 7)])
def test_i8_product_strides_and_alignment(pad, shift):
    gen = _gen(3)
    hold = torch.randint(-127, 128, (2 * 70 * (96 + pad) + shift,), generator=gen, device="cuda").to(torch.int8)
    w = hold.as_strided((2, 70, 96), (70 * (96 + pad), 96 + pad, 1), shift)
    x = torch.randint(-127, 128, (50 * (96 + pad) + shift,), generator=gen, device="cuda").to(torch.int8).as_strided((50, 96), (96 + pad, 1), shift)
    _check_i8(x, torch.rand(50, generator=gen, device="cuda"), w, torch.rand((2, 70), generator=gen, device="cuda"), [0, 20, 49], torch.float32)


@pytest.mark.parametrize("rows", (1, 40))
def test_i8_sums_stay_exact_at_the_longest_rows(rows):
    n = 131071
    q = torch.full((rows, n), -128, dtype=torch.int8, device="cuda")
    w = torch.full((1, 70, n), -128, dtype=torch.int8, device="cuda")
    w[0, 1::2] = 127
    q[:, 5], w[0, :, 7] = 3, 1
    ones = torch.ones(70, device="cuda")
    _check_i8(q, ones[:rows], w, ones[None], [0, rows], torch.float32, given=False)


# ---- handing out ----

def _slots(gen, tokens, top_k, masked):
    free = torch.rand(tokens, generator=gen, device="cuda") >= masked
    slots = torch.randperm(tokens * top_k, generator=gen, device="cuda")
    order = slots[free[slots // top_k]]
    position = torch.full((tokens * top_k,), -1, device="cuda")
    position[order] = torch.arange(len(order), device="cuda")
    order = torch.cat([order, torch.full((tokens * top_k - len(order),), -1, device="cuda")])
    return order.int(), position.reshape(tokens, top_k).int()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("weighted", (False, True))
@pytest.mark.parametrize("tokens,top_k,width,pad", [(1, 1, 1, 0), (1, 6, 520, 0), (50, 2, 33, 3), (300, 8, 1024, 0), (77, 32, 100, 4), (9, 3, 5000, 0)])
def test_hand_out_and_gradient(kind, weighted, tokens, top_k, width, pad):
    gen = _gen(tokens + width)
    order, position = _slots(gen, tokens, top_k, 0.3 if tokens > 1 else 0.0)
    x, drows = _inside((tokens, width), kind, pad, pad % 2), _inside((tokens * top_k, width), kind, pad, pad % 2)
    x.copy_(_normal(gen, tokens, width)), drows.copy_(_normal(gen, tokens * top_k, width))
    there = order >= 0
    drows[~there] = NAN
    weights = torch.rand((tokens, top_k), generator=gen, device="cuda") if weighted else None
    desc = tb.ExpertCombineDesc(tokens=tokens, rows=tokens * top_k, width=width, rows_stride=width + pad, out_stride=width + pad,
                                top_k=top_k, type=TYPES[kind])
    rows, dx = _inside((tokens * top_k, width), kind, pad, pad % 2), _inside((tokens, width), kind, pad, pad % 2)
    rows.fill_(3.0)
    dweights = torch.full((tokens, top_k), NAN, device="cuda")
    assert tb.tb_cuda_hand_out_experts_device(desc, x, order, weights, rows) == 1
    assert tb.tb_cuda_hand_out_experts_backward_device(desc, x, position, weights, drows, dx, dweights) == 1
    torch.cuda.synchronize()
    w = torch.ones((tokens, top_k), dtype=torch.float64, device="cuda") if weights is None else weights.double()
    slot = order[there].long()
    want = x.double()[slot // top_k] * w.flatten()[slot][:, None]
    check("rows", rows[there], want, U * want.abs() if weighted else 0 * want)
    assert (rows[~there] == 3).all()
    back = torch.where((position >= 0)[..., None], drows.double()[position.clamp(min=0).long()], torch.zeros((), dtype=torch.float64, device="cuda"))
    check("dx", dx, (back * w[..., None]).sum(1), (top_k + 1) * U * (back * w[..., None]).abs().sum(1))
    each = back * x.double()[:, None]
    # a lane sums at most width/32 + 8 terms, lanes and warps 13 more
    check("dweights", dweights, each.sum(2), (width / 32 + 24) * U * each.abs().sum(2))
    # either output alone
    alone = torch.empty_like(dweights)
    assert tb.tb_cuda_hand_out_experts_backward_device(desc, x, position, weights, drows, None, alone) == 1
    dx2 = torch.empty_like(dx).as_strided(dx.shape, dx.stride()) if pad == 0 else _inside((tokens, width), kind, pad, pad % 2)
    assert tb.tb_cuda_hand_out_experts_backward_device(desc, None, position, weights, drows, dx2, None) == 1
    torch.cuda.synchronize()
    assert torch.equal(alone, dweights) and torch.equal(dx2, dx)


def test_hand_out_is_what_the_combine_undoes():
    gen = _gen(4)
    order, position = _slots(gen, 64, 3, 0.0)
    x = _normal(gen, 64, 200, kind=torch.bfloat16)
    desc = tb.ExpertCombineDesc(tokens=64, rows=192, width=200, top_k=3, type=tb.TB_TYPE_BF16)
    rows, back = torch.empty((192, 200), device="cuda").bfloat16(), torch.empty_like(x)
    assert tb.tb_cuda_hand_out_experts_device(desc, x, order, None, rows) == 1
    third = torch.full((64, 3), 1 / 3, device="cuda")
    assert tb.tb_cuda_combine_experts_device(desc, rows, position, third, back) == 1
    torch.cuda.synchronize()
    check("back", back, x.double(), 4 * U * x.double().abs())


# ---- orthogonalised updates ----

QUINTIC = dict(a=3.4445, b=-4.7750, c=2.0315)


def _orthogonalise(g, out, steps=5, epsilon=1e-7, scale=1.0, **coefficients):
    b, m, n = g.shape
    desc = tb.OrthogonaliseDesc(matrices=b, rows=m, columns=n, in_matrix_stride=g.stride(0), in_row_stride=g.stride(1),
                                out_matrix_stride=out.stride(0), out_row_stride=out.stride(1), type=TYPES[g.dtype], steps=steps,
                                epsilon=epsilon, scale=scale, **{**QUINTIC, **coefficients})
    work = _work(tb.tb_cuda_orthogonalise_workspace(desc))
    assert tb.tb_cuda_orthogonalise_device(desc, g, out, work, torch.cuda.current_stream()) == 1
    _synchronised()


def _check_orthogonalise(g, out=None, steps=5, epsilon=1e-7, scale=1.0):
    out = torch.full(g.shape, NAN, device="cuda").to(g.dtype) if out is None else out
    before = g.clone()
    _orthogonalise(g, out, steps, epsilon, scale)
    want, error = ref.orthogonalise_error(before, steps, *QUINTIC.values(), epsilon, scale)
    check("update", out, want, error)


MATRICES = [(1, 1, 1), (2, 1, 9), (1, 7, 1), (3, 16, 33), (3, 33, 20), (2, 64, 64), (1, 100, 130), (8, 128, 256), (2, 256, 128),
            (1, 129, 129), (1, 257, 300), (2, 500, 300), (1, 515, 900), (1, 40, 3000), (1, 3001, 90)]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", MATRICES, ids=str)
def test_orthogonalise(shape, kind):
    _check_orthogonalise(_normal(_gen(sum(shape)), *shape, kind=kind, scale=0.02))


@pytest.mark.parametrize("steps,scale,epsilon", [(1, 1.0, 0.0), (2, -0.3, 1e-3), (9, 7.0, 1e-7)])
def test_orthogonalise_steps_and_scale(steps, scale, epsilon):
    _check_orthogonalise(_normal(_gen(steps), 2, 60, 90), steps=steps, scale=scale, epsilon=epsilon)


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_orthogonalise_strides_alignment_and_in_place(kind):
    for pad, shift in [(8, 0), (3, 1)]:
        g, out = _inside((2, 70, 50), kind, pad, shift), _inside((2, 70, 50), kind, pad + 2, shift)
        g.copy_(_normal(_gen(pad), 2, 70, 50))
        _check_orthogonalise(g, out)
        whole = torch.empty(0, device="cuda", dtype=kind).set_(out.untyped_storage())
        assert int(torch.isnan(whole).sum()) == whole.numel() - out.numel(), "written past the rows"
        _check_orthogonalise(g, g)


def test_orthogonalise_takes_any_size_of_gradient():
    """Squares that pass f32's range either way, low rank, a matrix of zeros, one that is not finite among others."""
    gen = _gen(12)
    g = _normal(gen, 6, 48, 80)
    g[0] *= 1e30
    g[1] *= 1e-30
    g[2] = _normal(gen, 48, 1) @ _normal(gen, 1, 80)
    g[3] = 0
    out = torch.empty_like(g)
    _orthogonalise(g, out, epsilon=0.0)
    want, error = ref.orthogonalise_error(g, 5, *QUINTIC.values(), 0.0, 1.0)
    check("update", out, want, error)
    assert (out[3] == 0).all()
    kept = out.clone()
    g[4, 1, 2] = float("inf")
    g[1, 0, 0] = NAN
    _orthogonalise(g, out, epsilon=0.0)
    assert torch.isnan(out[4]).all() and torch.isnan(out[1]).all()
    assert torch.equal(out[[0, 2, 3, 5]], kept[[0, 2, 3, 5]])


def test_orthogonalise_gives_the_same_bits():
    g = _normal(_gen(13), 3, 300, 200)
    first, again = torch.empty_like(g), torch.empty_like(g)
    _orthogonalise(g, first)
    for _ in range(3):
        _orthogonalise(g, again)
        assert torch.equal(first, again)


# ---- captured, on other streams, and together ----

def test_calls_are_captured_and_replayed_on_new_inputs():
    """Offsets, rows and weights change between replays; a second graph has a workspace of its own."""
    gen = _gen(14)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        rows, n, m = 400, 136, 200
        desc, x, w, dy, _ = _product_case(gen, rows, [0, 100, 300, 400], n, m, torch.bfloat16, False)
        off, work = _whole([0, 100, 300, 400]), _work(tb.tb_cuda_experts_product_workspace(desc))
        y, dx, dw = torch.empty((rows, m), device="cuda").bfloat16(), torch.empty((rows, n), device="cuda").bfloat16(), torch.empty_like(w)
        g, out = _normal(gen, 2, 90, 60), torch.empty((2, 90, 60), device="cuda")
        od = tb.OrthogonaliseDesc(matrices=2, rows=90, columns=60, type=0, steps=5, epsilon=1e-7, scale=1.0, **QUINTIC)
        owork = _work(tb.tb_cuda_orthogonalise_workspace(od))

        def run():
            assert tb.tb_cuda_experts_product_device(desc, x, w, off, y, work, torch.cuda.current_stream()) == 1
            assert tb.tb_cuda_experts_product_backward_device(desc, x, w, off, dy, dx, dw, work, torch.cuda.current_stream()) == 1
            assert tb.tb_cuda_orthogonalise_device(od, g, out, owork, torch.cuda.current_stream()) == 1

        run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed, offsets in [(1, [0, 0, 7, 400]), (2, [0, 399, 399, 399]), (3, [5, 50, 60, 61])]:
        gen = _gen(seed)
        x.copy_(_normal(gen, rows, n)), dy.copy_(_normal(gen, rows, m)), w.copy_(_normal(gen, 3, n, m)), off.copy_(_whole(offsets))
        g.copy_(_normal(gen, 2, 90, 60))
        y.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        used = torch.zeros(rows, dtype=torch.bool, device="cuda")
        used[offsets[0]:offsets[-1]] = True
        want, size = ref.product(x.double(), w.double(), offsets, False)
        check("y", y[used], want[used], ref.sum_error(n, size[used]))
        assert (y[~used] == 3).all()
        _, (dw_want, dw_size), depth = ref.product_backward(x.double(), w.double(), offsets, dy.double(), False)
        check("dw", dw, dw_want, ref.sum_error(depth, dw_size))
        o_want, o_error = ref.orthogonalise_error(g, 5, *QUINTIC.values(), 1e-7, 1.0)
        check("update", out, o_want, o_error)


def test_two_streams_at_once():
    gen = _gen(15)
    jobs = []
    for k in range(2):
        desc, x, w, dy, _ = _product_case(gen, 3000, [0, 1100, 3000], 512, 768, torch.bfloat16, k == 0)
        jobs.append((torch.cuda.Stream(), desc, x, w, torch.empty((3000, 768), device="cuda").bfloat16(),
                     _work(tb.tb_cuda_experts_product_workspace(desc))))
    off = _whole([0, 1100, 3000])
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, desc, x, w, y, work in jobs:
            assert tb.tb_cuda_experts_product_device(desc, x, w, off, y, work, stream) == 1
    for stream, *_ in jobs:
        assert tb.tb_cuda_synchronize(stream) == 1
    for k, (_, _, x, w, y, _) in enumerate(jobs):
        want, size = ref.product(x.double(), w.double(), [0, 1100, 3000], k == 0)
        check("y", y, want, ref.sum_error(512, size))


def test_product_over_2_31_elements():
    """The last expert's rows, far behind 2^31 elements of x and y, have the bits of a call of their own."""
    rows, n, m, tail = 4_300_000, 512, 520, 700
    gen = _gen(16)
    x = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    for part in x.split(1 << 19):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda"))
    w = _normal(gen, 2, m, n, kind=torch.bfloat16, scale=0.05)
    y, few = torch.empty((rows, m), dtype=torch.bfloat16, device="cuda"), torch.empty((tail, m), dtype=torch.bfloat16, device="cuda")
    for count, xs, ys, offsets in [(rows, x, y, [0, rows - tail, rows]), (tail, x[-tail:].clone(), few, [0, 0, tail])]:
        desc = tb.ExpertProductDesc(rows=count, experts=2, in_width=n, out_width=m, weight_order=tb.TB_WEIGHT_OUT_IN, type=tb.TB_TYPE_BF16)
        # 16-byte rows: nothing is laid out anew, the room for it is not touched
        assert tb.tb_cuda_experts_product_device(desc, xs, w, _whole(offsets), ys, torch.empty(16, dtype=torch.uint8, device="cuda")) == 1
    torch.cuda.synchronize()
    assert torch.equal(y[-tail:], few)
    del x, y
    torch.cuda.empty_cache()


def test_a_layer_of_experts_and_its_gradients():
    """Routing, handing out, two products, the combine, and back, as a learner uses them, against 64 bits."""
    gen = _gen(17)
    tokens, e, k, d, h = 150, 6, 2, 48, 80
    x, logits = _normal(gen, tokens, d), _normal(gen, tokens, e)
    up, down = _normal(gen, e, d, h, scale=d ** -0.5), _normal(gen, e, h, d, scale=h ** -0.5)
    dout = _normal(gen, tokens, d)
    route = tb.ExpertRouteDesc(tokens=tokens, experts=e, top_k=k, groups=1, top_groups=1, group_best=1, type=0, score=tb.TB_SCORE_SOFTMAX,
                               renormalise=1, weight_scale=1.0)
    whole = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, offsets, order, position, weights = whole(tokens, k), whole(e + 1), whole(tokens * k), whole(tokens, k), torch.empty((tokens, k), device="cuda")
    new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    r = tokens * k
    assert tb.tb_cuda_route_experts_device(route, logits, None, ids, weights, offsets, order, position, _work(tb.tb_cuda_route_experts_workspace(route))) == 1
    comb = tb.ExpertCombineDesc(tokens=tokens, rows=r, width=d, top_k=k, type=0)
    pu, pd = (tb.ExpertProductDesc(rows=r, experts=e, in_width=i, out_width=o, weight_order=tb.TB_WEIGHT_IN_OUT, type=0) for i, o in ((d, h), (h, d)))
    wu, wd = (_work(tb.tb_cuda_experts_product_workspace(p)) for p in (pu, pd))
    rows, u, out_rows, out = new(r, d), new(r, h), new(r, d), new(tokens, d)
    assert tb.tb_cuda_hand_out_experts_device(comb, x, order, None, rows) == 1
    assert tb.tb_cuda_experts_product_device(pu, rows, up, offsets, u, wu) == 1
    act = torch.tanh(u)
    assert tb.tb_cuda_experts_product_device(pd, act, down, offsets, out_rows, wd) == 1
    assert tb.tb_cuda_combine_experts_device(comb, out_rows, position, weights, out) == 1
    d_rows, dweights, dact, ddown, dx_rows, dup, dx = new(r, d), new(tokens, k), new(r, h), new(e, h, d), new(r, d), new(e, d, h), new(tokens, d)
    assert tb.tb_cuda_combine_experts_backward_device(comb, out_rows, position, weights, dout, d_rows, dweights) == 1
    assert tb.tb_cuda_experts_product_backward_device(pd, act, down, offsets, d_rows, dact, ddown, wd) == 1
    du = dact * (1 - act * act)
    assert tb.tb_cuda_experts_product_backward_device(pu, rows, up, offsets, du, dx_rows, dup, wu) == 1
    assert tb.tb_cuda_hand_out_experts_backward_device(comb, None, position, None, dx_rows, dx, None) == 1
    torch.cuda.synchronize()
    x64, up64, down64 = (v.double().requires_grad_() for v in (x, up, down))
    w64 = torch.softmax(logits.double(), 1).gather(1, ids.long())
    w64 = (w64 / w64.sum(1, keepdim=True)).requires_grad_()
    each = torch.einsum("tkh,tkhd->tkd", torch.tanh(torch.einsum("td,tkdh->tkh", x64, up64[ids.long()])), down64[ids.long()])
    want = (each * w64[..., None]).sum(1)
    grads = torch.autograd.grad(want, (x64, up64, down64, w64), dout.double())
    # a few dozen f32 roundings of values of order one, each below 1e-7, through two layers of 80 terms
    torch.testing.assert_close(out.double(), want.detach(), rtol=1e-5, atol=1e-5)
    for got, g in zip((dx, dup, ddown, dweights), grads):
        torch.testing.assert_close(got.double(), g, rtol=1e-5, atol=2e-5 * float(g.abs().max()))


# ---- refusals where a call that is not refused returns 1 ----

CALLS = {
    "hand_out": (tb.tb_cuda_hand_out_experts_device, tb.ExpertCombineDesc(tokens=20, rows=40, width=32, top_k=2, type=0),
                 "x order weights ROWS", []),
    "hand_out_backward": (tb.tb_cuda_hand_out_experts_backward_device, tb.ExpertCombineDesc(tokens=20, rows=40, width=32, top_k=2, type=0),
                          "x position weights drows DX DWEIGHTS", []),
    "product": (tb.tb_cuda_experts_product_device, tb.ExpertProductDesc(rows=40, experts=2, in_width=32, out_width=48, type=0),
                "x weight offsets Y WORK", []),
    "product_backward": (tb.tb_cuda_experts_product_backward_device,
                         tb.ExpertProductDesc(rows=40, experts=2, in_width=32, out_width=48, type=0),
                         "x weight offsets dy DX DWEIGHT WORK", []),
    "quantise": (tb.tb_cuda_quantise_rows_device, tb.QuantiseDesc(rows=40, width=32, type=0), "x Q SCALE", []),
    "i8": (tb.tb_cuda_experts_product_i8_device, tb.ExpertProductI8Desc(rows=40, experts=2, in_width=32, out_width=48, type=0),
           "q q_scale weight weight_scale offsets Y WORK", []),
    "orthogonalise": (tb.tb_cuda_orthogonalise_device,
                      tb.OrthogonaliseDesc(matrices=2, rows=20, columns=30, type=0, steps=2, epsilon=1e-7, scale=1.0, **QUINTIC),
                      "g OUT WORK", [("g", "OUT")]),
}


@pytest.mark.parametrize("name", CALLS)
def test_outputs_on_inputs_are_refused(name):
    call, desc, names, stated = CALLS[name]
    names = names.split()
    buffers = {n: torch.zeros(1 << 18, device="cuda") for n in names}

    def run(**change):
        return call(desc, *[{**buffers, **change}[n] for n in names])

    assert run() == 1
    torch.cuda.synchronize()
    for n in names:
        for other in names:
            if n == other or not n.isupper() or (other, n) in stated:
                continue
            assert run(**{n: buffers[other]}) == 0, (n, other)
    for other, n in stated:
        assert run(**{n: buffers[other]}) == 1, (n, other)
    torch.cuda.synchronize()
