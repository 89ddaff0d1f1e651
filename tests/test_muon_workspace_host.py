"""Workspace where memory is short: the products take less and pass through it more often."""
import pytest
import torch

from hybridagent_b200 import muon


@pytest.mark.parametrize("free,sizes", [(1000, [1000]), (999, [1000, 500]), (200, [1000, 500, 250, 125]), (101, [1000, 500, 250, 125, 101]),
                                        (100, None)])
def test_less_is_taken_where_memory_is_short(monkeypatch, free, sizes):
    asked = []

    def empty(size, **kw):
        asked.append(size)
        if size > free:
            raise torch.OutOfMemoryError("no room")
        return size

    monkeypatch.setattr(muon.torch, "empty", empty)
    if sizes is None:  # not even the least
        with pytest.raises(torch.OutOfMemoryError):
            muon._workspace(1000, 101, torch.device("cuda"))
        assert asked[-1] == 101
    else:
        assert muon._workspace(1000, 101, torch.device("cuda")) == sizes[-1]
        assert asked == sizes
