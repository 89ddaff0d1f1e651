"""Orthogonalisation of matrices that are low-rank, nearly so, or fall off quickly, over few and many steps.

Bounds (2-norm, relative), all in units of what rounding the result to bf16 takes, r = 0.42 * 2^-8 in the root mean square
(half a step spread evenly over the mantissas; an fp16 value's is r / 8).  X in a single fp16 plane is off by r / 8, and
the steps behind it multiply that by at most 12 in directions that X has not: 1.5 r.  A step's Gram matrix and its factor,
each off by r / 8, turn the singular vectors by 3.45 / 0.68 of it (a factor is at most 3.45, a singular value near one is
multiplied by 0.68 or more): 0.63 r each, ten of them in five steps.  Added as independent, with the result's own
rounding: sqrt(1 + 1.5^2 + 10 * 0.63^2) = 2.7.  Where a pair of steps runs as one, its first two are multiplied
by 3.45 once more: sqrt(1 + 1.5^2 + 8 * 0.63^2 + 2 * (3.45 * 0.63)^2) = 4.0.

More steps add as many roundings each.  What is off in directions that X does not have is multiplied by all steps that
follow, in any arithmetic; in those the kernel is limited by its accumulators.  The matrix unit adds 16 products and the
accumulator at a time, aligned to the largest of them and cut off at its last place, u = 2^-23 of it at most: 17 errors
spread over u have the deviation u sqrt(17 / 12) / mantissa, 0.88 u in the root mean square (mantissas of
even logarithm), and what cutting takes from the accumulator itself, u / 2, differs between elements by 0.14 u / 2.  Over the m / 16
additions of a step on the shorter side m that is u sqrt(0.88^2 m / 16 + (0.072 m / 16)^2), and over all steps, with X
no larger than 1.2 times the result, half the product of all gains times it; the bound is twice that."""
import math

import pytest

from hybridagent_b200 import muon

pytestmark = pytest.mark.gpu

KINDS = ["rank1", "rank4", "rank32", "rank4_and_noise", "power_law", "four_decades"]


def spectrum(kind, rows, cols, seed=0):
    """A matrix with that spectrum, in 64 bits."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float64)

    if kind.startswith("rank") and kind[4:].isdigit():
        rank = int(kind[4:])
        return normal(rows, rank) @ normal(rank, cols)
    if kind == "rank4_and_noise":
        return normal(rows, 4) @ normal(4, cols) + 2e-3 * normal(rows, cols)
    m = min(rows, cols)
    left, right = (torch.linalg.qr(normal(n, m))[0] for n in (rows, cols))
    k = torch.arange(m, device="cuda", dtype=torch.float64)
    return left * (1 / (k + 1) if kind == "power_law" else 10.0 ** (-4 * k / m)) @ right.mT


def definition(x, rows):
    x = x.double()
    if x.shape[0] > x.shape[1]:
        return definition(x.mT, rows).mT
    x = x / x.norm()
    for a, b, c in rows:
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def check(x, rows, merged):
    from hybridagent_b200 import orthogonalize
    x = x.float()
    want = definition(x, rows)
    bound = (4.0 if merged else 2.7) * math.sqrt(max(len(rows), 5) / 5)
    adds = min(x.shape) / 16
    brought_up = math.prod(abs(row[0]) for row in rows) * 2.0 ** -23 * math.hypot(0.88 * math.sqrt(adds), 0.072 * adds)
    got = off(orthogonalize(x, steps=len(rows), coefficients=rows), want)
    assert got <= bound * off(want.bfloat16(), want) + brought_up


# (rows, cols), and whether pairs of steps are merged
SHAPES = [((300, 400), False), ((400, 300), False), ((200, 900), False), ((300, 500), True), ((1100, 330), True),
          ((704, 2816), True), ((1700, 800), True), ((1024, 2048), True), ((700, 1900), True), ((5000, 2100), True)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,merged", SHAPES, ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else "")
def test_five_steps(shape, merged, kind):
    check(spectrum(kind, *shape, seed=sum(shape)), [muon.COEFFICIENTS] * 5, merged)


@pytest.mark.parametrize("steps", [6, 8, 10])
@pytest.mark.parametrize("kind", ["rank4", "rank32", "rank4_and_noise", "four_decades"])
@pytest.mark.parametrize("shape,merged", SHAPES, ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else "")
def test_more_steps_do_not_bring_up_noise(shape, merged, kind, steps):
    check(spectrum(kind, *shape, seed=sum(shape)), [muon.COEFFICIENTS] * steps, merged)


@pytest.mark.parametrize("shape,merged", SHAPES, ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else "")
def test_sixteen_cubic_steps(shape, merged):
    """Steps of small gain: 1.5 each, 657 together."""
    check(spectrum("rank4", *shape, seed=sum(shape)), [(1.5, -0.5, 0.0)] * 16, merged)


@pytest.mark.parametrize("shape", [(1, 1), (1, 40), (37, 1), (2, 3), (5, 7), (31, 33), (64, 96), (128, 128), (128, 1000), (1000, 17),
                                   (16, 9000), (300, 400)], ids=lambda s: "x".join(map(str, s)))
def test_steps_of_large_gain(shape):
    """A first step that multiplies by 13, more than the kernel of short sides takes: those run like long ones, and what a
    single plane's rounding would grow to does not show."""
    import torch
    rows = [(13.0, -30.0, 17.5), (1.2, -0.1, 0.0)]
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = torch.randn(3, *shape, generator=gen, device="cuda")
    from hybridagent_b200 import orthogonalize
    y = orthogonalize(x, steps=2, coefficients=rows)
    for k in range(3):
        want = definition(x[k], rows)
        # per step: Gram matrix and factor, r / 8 of 30 + 17.5 and 13 at most, on singular values multiplied by 0.5 or more
        bound = off(want.bfloat16(), want) + 2 * (47.5 + 13) / 0.5 * 0.42 * 2.0 ** -11
        assert off(y[k], want) <= bound
