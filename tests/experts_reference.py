"""The experts' operators in 64 bits (torch on any device), written from the formulas of
include/turbinator/training/cuda_learner.h, with bounds on what the kernels' arithmetic may be off.

U is the unit roundoff of f32.  The tensor cores' own sums are not documented to the last bit: an instruction that adds
16 products (32 of 8 bits, exactly) to an accumulator is taken to be off by no more than 4 U of the magnitudes summed so
far.  tests/learner_reference.py has what a result's storing adds (`stored`, `check`)."""
from __future__ import annotations

import torch

from tests.learner_reference import U


def sum_error(depth, magnitude, f32=False):
    """Bound on a sum of `depth` products of the tensor cores, sum of magnitudes `magnitude`.  f32 operands are three
    parts of 8 bits: six of nine pairs of parts, what is left out is below 2^-24 + 2^-25 of a product, twice that with
    the parts' own rounding."""
    steps = depth / 16 + 2
    if not f32:
        return 4 * U * steps * magnitude
    return (4 * U * 6 * steps + 4 * U) * magnitude


def runs(offsets, rows):
    ends = [min(max(int(o), 0), rows) for o in offsets]
    return [(e, slice(a, z)) for e, (a, z) in enumerate(zip(ends, ends[1:])) if z > a]


def product(x, w, offsets, turned):
    """y [rows, out] (NaN in rows of no expert) and the sums of magnitudes."""
    y = torch.full((x.shape[0], w.shape[1] if turned else w.shape[2]), float("nan"), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    for e, r in runs(offsets, x.shape[0]):
        m = w[e].T if turned else w[e]
        y[r], size[r] = x[r] @ m, x[r].abs() @ m.abs()
    return y, size


def product_backward(x, w, offsets, dy, turned):
    """dx (NaN in rows of no expert), dw and the sums of magnitudes of both, and each expert's rows."""
    dx, dx_size = product(dy, w.transpose(1, 2), offsets, turned)
    dw, dw_size = torch.zeros_like(w), torch.zeros_like(w)
    depth = torch.zeros((w.shape[0], 1, 1), dtype=torch.float64, device=x.device)
    for e, r in runs(offsets, x.shape[0]):
        left, right = (dy[r], x[r]) if turned else (x[r], dy[r])
        dw[e], dw_size[e] = left.T @ right, left.abs().T @ right.abs()
        depth[e] = r.stop - r.start
    return (dx, dx_size), (dw, dw_size), depth


def quantise(x):
    """q and scale of rows, each operation rounded in f32 as the header states it."""
    x = x.float()
    most = x.abs().amax(1)
    up = (torch.ones_like(most) / most) * 127
    bad = ~torch.isfinite(x).all(1)
    none = bad | ~torch.isfinite(up)
    q = torch.round(x * up[:, None]).masked_fill(none[:, None], 0).to(torch.int8)
    scale = torch.where(none, torch.zeros_like(most), most / torch.full_like(most, 127))
    return q, scale.masked_fill(bad, float("nan"))


def orthogonalise(g, steps, a, b, c, epsilon, scale, noise=None):
    """The polynomial's steps; `noise(value, magnitude)` is added to what is rounded on the way."""
    noise = noise or (lambda v, _: v)
    x = g.double()
    norm = torch.linalg.matrix_norm(x)[:, None, None]
    x = torch.where(norm > 0, x / (norm + epsilon), x)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = noise(x, x.abs())
    for _ in range(steps):
        t = x.transpose(1, 2)
        gram = noise(x @ t, x.abs() @ t.abs())
        poly = b * gram + c * noise(gram @ gram, gram.abs() @ gram.abs())
        poly = noise(poly, poly.abs())
        x = a * x + noise(poly @ x, poly.abs() @ x.abs())
        x = noise(x, x.abs())
    return scale * (x.transpose(1, 2) if tall else x)


def orthogonalise_error(g, steps, a, b, c, epsilon, scale):
    """Bound on each element.  Every kept value is rounded to 22 bits (2^-22 of itself, or 2^-37), every product leaves
    out 2^-21 of its magnitudes and adds them in sums of 64 of k: 4 instructions of three products each, 4 U of the
    magnitudes each, so 2^-22 (2 + 12) < 2^-18 of them at worst.  The steps carry these errors on linearly; the
    definition with errors of that size and random signs says how far, and 16 times the root mean square of what it
    does in four runs covers every element."""
    gen = torch.Generator(device=g.device)
    gen.manual_seed(99)

    def noise(v, magnitude):
        sign = torch.randint(0, 2, v.shape, generator=gen, device=v.device) * 2.0 - 1
        sign = torch.tril(sign) + torch.tril(sign, -1).transpose(1, 2) if v.shape[1] == v.shape[2] else sign
        return v + sign * (2.0 ** -18 * magnitude + 2.0 ** -37)

    want = orthogonalise(g, steps, a, b, c, epsilon, scale)
    off = [(orthogonalise(g, steps, a, b, c, epsilon, scale, noise) - want).square() for _ in range(4)]
    mean = torch.stack(off).mean((0, 2, 3)).sqrt()[:, None, None]
    return want, 16 * mean + 8 * U * want.abs()
