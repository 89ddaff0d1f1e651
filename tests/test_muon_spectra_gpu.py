"""Orthogonalisation of matrices that are low-rank, nearly so, or fall off quickly.

Bounds (2-norm, relative), all in units of what rounding the result to bf16 takes, r = 0.42 * 2^-8 in the root mean square
(half a step spread evenly over the mantissas; an fp16 value's is r / 8).  X in a single fp16 plane is off by r / 8, and
the steps behind it multiply that by at most 12 in directions that X has not: 1.5 r.  A step's Gram matrix and its factor,
each off by r / 8, turn the singular vectors by 3.45 / 0.68 of it (a factor is at most 3.45, a singular value near one is
multiplied by 0.68 or more): 0.63 r each, ten of them in five steps.  Added as independent, with the result's own
rounding: sqrt(1 + 1.5^2 + 10 * 0.63^2) = 2.7.  Where a pair of steps runs as one, its first two are multiplied
by 3.45 once more: sqrt(1 + 1.5^2 + 8 * 0.63^2 + 2 * (3.45 * 0.63)^2) = 4.0."""
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
    got = off(orthogonalize(x, steps=len(rows), coefficients=rows), want)
    assert got <= (4.0 if merged else 2.7) * off(want.bfloat16(), want)


# (rows, cols), and whether pairs of steps are merged
SHAPES = [((300, 400), False), ((400, 300), False), ((200, 900), False), ((300, 500), True), ((1100, 330), True),
          ((704, 2816), True), ((1700, 800), True), ((1024, 2048), True), ((700, 1900), True), ((5000, 2100), True)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,merged", SHAPES, ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else "")
def test_five_steps(shape, merged, kind):
    check(spectrum(kind, *shape, seed=sum(shape)), [muon.COEFFICIENTS] * 5, merged)
