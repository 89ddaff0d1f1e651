"""Orthogonalisation of matrices with very long sides, whose Gram matrices are sums of up to millions of products.

The matrix unit cuts its sums off by up to 2^-23 of them at each addition of 16 products, 2^-24 in the mean and always
towards zero.  Added up in parts of 2048 additions, a Gram matrix is off by 2048 * 2^-24 = 1.2e-4; a step takes that to
X 4.8 (|b|) times at most: 5.9e-4, five times, added as independent to what rounding to bf16 takes, 1.66e-3:
sqrt(1.66^2 + 5 * 0.59^2) = 2.1e-3, which is less than 1.5 times the rounding."""
import pytest

from hybridagent_b200 import muon

pytestmark = pytest.mark.gpu

PIECE = 1 << 18


def factor(x):
    """The product of all steps' factors and 1 / norm in 64 bits, from the Gram matrix of x (rows <= cols), piece by piece."""
    import torch
    gram = torch.zeros(x.shape[0], x.shape[0], dtype=torch.float64, device="cuda")
    for k in range(0, x.shape[1], PIECE):
        p = x[:, k:k + PIECE].double()
        gram += p @ p.mT
    norm = gram.trace().sqrt()
    gram /= norm ** 2
    one = left = torch.eye(x.shape[0], dtype=torch.float64, device="cuda")
    a, b, c = muon.COEFFICIENTS
    for _ in range(5):
        q = a * one + b * gram + c * (gram @ gram)
        left = q @ left
        gram = q @ gram @ q
    return left / norm


def off_and_rounding(y, x, left):
    """Relative errors of y, and of the exact result as bf16."""
    error = rounding = size = 0.0
    for k in range(0, x.shape[1], PIECE):
        want = left @ x[:, k:k + PIECE].double()
        error += float((y[:, k:k + PIECE].double() - want).square().sum())
        rounding += float((want.bfloat16().double() - want).square().sum())
        size += float(want.square().sum())
    return (error / size) ** 0.5, (rounding / size) ** 0.5


@pytest.mark.parametrize("rows,cols", [(160, 32768), (160, 32776), (160, 65537), (300, 200000), (200000, 300), (160, 1000000), (1000, 70000),
                                       (131100, 520), (64, 4000000), (4000000, 50), (16, 9000000), (1, 16000000), (128, 140000),
                                       (140000, 128), (3, 131073 * 8)])
def test_long_sides(rows, cols):
    import torch
    from hybridagent_b200 import orthogonalize
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    y = orthogonalize(x)
    assert torch.equal(y, orthogonalize(x))
    if rows > cols:
        x, y = x.mT, y.mT
    error, rounding = off_and_rounding(y, x, factor(x))
    assert error <= 1.5 * rounding


def test_long_batches_of_several_shapes():
    """Matrices that share a launch, in a Muon step, with sides around those of the parts."""
    import torch
    from hybridagent_b200 import ZeroOneMuon
    shapes = [(140, 40000), (140, 40000), (66000, 150), (150, 3000), (300, 32768), (70, 50000)]
    params = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in shapes]
    opt = ZeroOneMuon([{"params": params, "lr": 1.0}], rank=0, world_size=1, adjust_lr=None, momentum=0.0)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda") * 1e-3
    opt.step()
    for p in params:
        g, w = (p.grad, p.detach()) if p.shape[0] <= p.shape[1] else (p.grad.mT, p.detach().mT)
        error, rounding = off_and_rounding(-w, g, factor(g))
        assert error <= 1.5 * rounding


@pytest.mark.parametrize("shape", [(2, 2000, 40000), (1, 36000, 2100), (3, 300, 33000), (2, 70000, 140)],
                         ids=lambda s: "x".join(map(str, s)))
def test_long_batches_alone_and_replayed(shape):
    """On single CTAs and on pairs, as a graph too, whose second replay finds the first one's sums in the workspace."""
    import torch
    from hybridagent_b200 import orthogonalize
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = torch.randn(shape, generator=gen, device="cuda").bfloat16()
    y = orthogonalize(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = orthogonalize(x)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    for k in range(shape[0]):
        g, w = (x[k].float(), y[k]) if shape[1] <= shape[2] else (x[k].float().mT, y[k].mT)
        error, rounding = off_and_rounding(w, g, factor(g))
        assert error <= 1.5 * rounding
