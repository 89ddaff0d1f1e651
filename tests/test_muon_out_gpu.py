"""orthogonalize's result as a tensor of the caller."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(4, 64, 96), (2, 300, 401)], ids=lambda s: "x".join(map(str, s)))
def test_autograd_sees_that_out_was_written(shape):
    """A product that saved `out` for its backward pass refuses it once the values are others."""
    import torch
    from hybridagent_b200 import orthogonalize
    x = torch.randn(shape, device="cuda")
    out = torch.ones(shape, dtype=torch.bfloat16, device="cuda")
    weight = torch.randn(shape, device="cuda", requires_grad=True)
    loss = (weight * out).sum()
    version = out._version
    assert orthogonalize(x, out=out) is out
    assert out._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    (weight * out).sum().backward()
    assert torch.equal(weight.grad, out.float())
    with torch.inference_mode():
        inner = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(orthogonalize(x, out=inner), out)


def test_a_transposed_view_gives_a_transposed_view():
    import torch
    from hybridagent_b200 import orthogonalize
    x = torch.randn(3, 70, 50, device="cuda")
    y = orthogonalize(x.mT)
    assert y.shape == (3, 50, 70) and y.mT.is_contiguous() and torch.equal(y.mT, orthogonalize(x))
    out = torch.empty(3, 50, 70, dtype=torch.bfloat16, device="cuda")
    z = orthogonalize(x.mT, out=out)  # laid out as the caller wants it
    assert z is out and float((z.double() - y.double()).norm() / y.double().norm()) <= 2.0 ** -8
