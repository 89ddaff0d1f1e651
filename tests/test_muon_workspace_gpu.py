"""Calls where the device has little memory left."""
import pytest

from hybridagent_b200 import muon

pytestmark = pytest.mark.gpu


@pytest.fixture
def little_memory(monkeypatch):
    """Limits what torch.empty gives in one piece, as a function of that many bytes."""
    import torch
    real = torch.empty

    def limit(most):
        def empty(*size, **kw):
            if kw.get("dtype") is torch.uint8 and size[0] > most:
                raise torch.OutOfMemoryError("CUDA out of memory")
            return real(*size, **kw)
        monkeypatch.setattr(torch, "empty", empty)

    return limit


def test_orthogonalize(little_memory):
    import torch
    from hybridagent_b200 import orthogonalize
    x = torch.randn(40, 300, 500, device="cuda").bfloat16()
    want = orthogonalize(x)
    all_of_it = muon._workspace_bytes(40, 300, 500)
    out = torch.empty_like(x)
    little_memory(all_of_it // 2)
    assert orthogonalize(x, out=out) is out
    # (parts of a batch may take tiles of another size: another order of the same sums)
    assert float((out.double() - want.double()).norm() / want.double().norm()) <= 4e-3


def test_the_optimizer(little_memory):
    import torch
    from hybridagent_b200 import ZeroOneMuon
    params = [torch.nn.Parameter(torch.randn(600, 900, device="cuda").bfloat16() * 0.02) for _ in range(30)]
    for p in params:
        p.grad = torch.randn_like(p)
    before = [p.detach().clone() for p in params]
    little_memory(muon._workspace_bytes(10, 600, 900))
    opt = ZeroOneMuon([{"params": params, "lr": 1e-2}], rank=0, world_size=1)
    assert muon._workspace_bytes(1, 600, 900) <= opt._muon_ws.numel() <= muon._workspace_bytes(10, 600, 900)
    opt.clip_grad_norm(1.0)
    opt.step()
    assert opt.state_dict()["step_count"] == 1
    assert all(not torch.equal(a, b) for a, b in zip(before, params))
