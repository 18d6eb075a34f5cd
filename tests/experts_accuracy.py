"""How far the experts' operators' f32 results may lie from 64 bits on random data, by the kernels' own rule: what each
plane, each left-out product and each sum may be off, with signs that fall as they may.  A root mean square of many
elements is compared, so that a plane, a product of planes or a sum that is not taken as it should be shows.

U is the unit roundoff of f32.  A stage is 64 of k: four instructions of 16 for each pair of planes.  What the tensor
cores hold may be off by 4 U of it in each instruction; of the four of the first planes, where all of it is there,
the partial sums are sqrt(1/4), sqrt(2/4), .. of the stage's: 4 U (0.5 + 0.71 + 0.87 + 1) = 12.3 U, below 13 U of a stage,
the instructions of smaller planes included.  Stages are independent, and each one's addition in f32 is off by U / 2 of the
sum so far: 13 U + sqrt(stages / 2) U / 2 of the root of the sum of squares of the products."""
from __future__ import annotations

import math

import torch

from tests.learner_reference import U


def size(x, t):
    """Root of the sum of squares of the products that x @ t sums: their sum's own size, where signs are random."""
    return (x.square() @ t.square()).sqrt()


def sum_error(depth):
    """Of `size`."""
    stages = math.ceil(depth / 64)
    return (13 + 0.5 * math.sqrt(stages / 2)) * U


def rms(v):
    return float(v.double().square().mean().sqrt())


def update_with_errors(g, steps, a, b, c, epsilon, scale):
    """The orthogonalised update where everything kept is rounded to 22 bits (2^-22 of itself at most, and 2^-48) and
    every product carries its sum's error, of its sum as well as of its size, since a sum of squares has no random signs."""
    gen = torch.Generator(device=g.device)
    gen.manual_seed(98)

    def sign(v):
        s = torch.randint(0, 2, v.shape, generator=gen, device=v.device) * 2.0 - 1
        return torch.tril(s) + torch.tril(s, -1).transpose(1, 2) if v.shape[1] == v.shape[2] else s

    def kept(v):
        return v + sign(v) * (2.0 ** -22 * v.abs() + 2.0 ** -48)

    def product(x, t):
        v = x @ t
        return v + sign(v) * sum_error(x.shape[2]) * (size(x, t) + v.abs())

    x = g.double()
    x = x / (torch.linalg.matrix_norm(x)[:, None, None] + epsilon)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = kept(x)
    for _ in range(steps):
        gram = kept(product(x, x.transpose(1, 2)))
        poly = kept(b * gram + c * product(gram, gram))
        x = kept(a * x + product(poly, x))
    return scale * (x.transpose(1, 2) if tall else x)


def update_in_f32(g, steps, a, b, c, epsilon, scale):
    """The same in plain f32 arithmetic."""
    x = g.float()
    x = x / (torch.linalg.matrix_norm(x)[:, None, None] + epsilon)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    for _ in range(steps):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return scale * (x.transpose(1, 2) if tall else x)
