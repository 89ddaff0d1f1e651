"""The Muon step's stores into peers' copies of the parameters, emulated by buffers on this GPU."""
import ctypes

import numpy as np
import pytest

from hybridagent_b200 import _lib, muon

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(48, 72), (300, 280), (37, 53)])
@pytest.mark.parametrize("code,changed_only", [(1, 0), (1, 1), (2, 0), (2, 1)])
def test_a_peer_receives_the_changed_sectors_and_nothing_else(rows, cols, code, changed_only):
    """The peers' buffers start with bits that no update gives: what is stored there shows."""
    import torch
    dt = {1: torch.bfloat16, 2: torch.float16}[code]
    numel, n_peers, guard = rows * cols, 2, 64
    room = guard + (numel + 63) // 64 * 64 + guard
    gen = torch.Generator(device="cuda").manual_seed(rows)
    master = torch.randn(rows, cols, generator=gen, device="cuda") * 0.02
    grad = torch.randn(rows, cols, generator=gen, device="cuda").to(dt)
    moment = torch.zeros(rows, cols, device="cuda")
    copies = torch.full((1 + n_peers, room), -1, dtype=torch.int16, device="cuda")  # NaN
    here = copies[0, guard:guard + numel].view(dt)
    here.copy_(master.reshape(-1).to(dt))
    before = here.clone()
    tab = np.zeros(1, dtype=_lib.TENSOR_DTYPE)
    for name, value in (("grad", grad.data_ptr()), ("master", master.data_ptr()), ("exp_avg", moment.data_ptr()),
                        ("param", here.data_ptr()), ("numel", numel), ("decay", 1.0), ("neg_lr", -1e-5)):
        tab[name] = value
    peers = _lib.Peers()
    peers.n = n_peers
    for k in range(n_peers):
        peers.delta[k] = copies[1 + k].data_ptr() - copies[0].data_ptr()
    sc, ns = _lib.MuonScalars(0.95, 0.05, 1, 0, 0, 1.0), muon._ns_params(5, muon.COEFFICIENTS, 1e-7)
    size = muon._workspace_bytes(1, rows, cols)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    shapes = np.asarray([[rows, cols]], dtype=np.int64)
    _lib.call("ha_muon_step", _lib.np_ptr(tab), _lib.np_ptr(shapes), 1, code, ctypes.byref(sc), ctypes.byref(ns), changed_only,
              ctypes.byref(peers), count.data_ptr(), None, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(here, master.reshape(-1).to(dt))
    for k in range(1 + n_peers):  # nothing outside the tensor
        assert (copies[k, :guard] == -1).all() and (copies[k, guard + numel:] == -1).all()
    moved = here.view(torch.int16) != before.view(torch.int16)
    whole = numel // 16 * 16
    sectors = moved[:whole].view(-1, 16).any(1)
    assert 0 < int(sectors.sum()) and (not changed_only or int(sectors.sum()) < sectors.numel())
    if not changed_only:
        sectors[:] = True
    for k in range(1, 1 + n_peers):
        peer = copies[k, guard:guard + numel]
        stored = peer[:whole].view(-1, 16)
        assert torch.equal(stored[sectors], here[:whole].view(torch.int16).view(-1, 16)[sectors])
        assert (stored[~sectors] == -1).all()
        tail, moved_tail = peer[whole:], moved[whole:]
        assert torch.equal(tail[moved_tail], here[whole:].view(torch.int16)[moved_tail])
        assert ((tail == -1) | (tail == here[whole:].view(torch.int16))).all()
