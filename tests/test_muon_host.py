"""Muon on the host (no GPU): arguments that are refused, the workspace's size, and the layout with
matrices and other tensors in classes of their own."""
import ctypes

import numpy as np
import pytest
import torch

from hybridagent_b200 import ZeroOneMuon, _lib, layout, muon, orthogonalize


def _ns(steps=5, coefficients=muon.COEFFICIENTS, eps=1e-7):
    return muon._ns_params(steps, coefficients, eps)


def _bytes(batch, rows, cols):
    out = ctypes.c_size_t(0)
    _lib.call("ha_orthogonalize_workspace", batch, rows, cols, ctypes.byref(out))
    return out.value


def test_workspace_grows_with_the_batch_and_holds_the_planes():
    for rows, cols in ((1, 1), (64, 96), (256, 512), (1000, 1537), (4096, 12288), (17408, 5120)):
        one, two, many = (_bytes(n, rows, cols) for n in (1, 2, 40))
        assert _bytes(0, rows, cols) == one < two < many
        assert many < 41 * one
        assert one > 3 * 2 * rows * cols  # at least the high planes before and after a step, and the low plane
        assert _bytes(10**9, rows, cols) == _bytes(4096, rows, cols)  # the most that pass at once
    for bad in ((0, 5), (5, 0), (-1, 4), (1 << 25, 4), (1 << 24, 1 << 20)):
        with pytest.raises(_lib.HAError, match="matrices of"):
            _bytes(1, *bad)
    with pytest.raises(_lib.HAError, match="batch"):
        _bytes(-1, 4, 4)
    with pytest.raises(_lib.HAError, match="NULL"):
        _lib.call("ha_orthogonalize_workspace", 1, 4, 4, None)


# addresses that are never read: every call here is refused before a launch
SRC, DST, WS = 1 << 20, 1 << 21, 1 << 22


def _orthogonalize(src=SRC, code=_lib.HA_BF16, dst=DST, batch=1, rows=64, cols=96, ns=None, ws=WS, size=None):
    size = _bytes(1, rows, cols) if size is None else size
    _lib.call("ha_orthogonalize", src, code, dst, batch, rows, cols, ctypes.byref(_ns() if ns is None else ns), ws, size,
              None)


@pytest.mark.parametrize("kw,message", [
    (dict(code=7), "dtype"), (dict(code=_lib.HA_F64), "dtype"), (dict(batch=-1), "batch"), (dict(src=None), "NULL"),
    (dict(dst=None), "NULL"), (dict(src=SRC + 1), "misaligned"), (dict(src=SRC + 2, code=_lib.HA_F32), "misaligned"),
    (dict(dst=DST + 1), "misaligned"), (dict(ws=None), "256-byte"), (dict(ws=WS + 16), "256-byte"),
    (dict(size=1000), "one matrix needs"), (dict(size=0), "one matrix needs"),
    (dict(ns=_ns(eps=0.0)), "eps"), (dict(ns=_ns(eps=float("nan"))), "eps"), (dict(ns=_ns(eps=1e31)), "eps"),
    (dict(ns=_ns(coefficients=(70.0, 0.0, 0.0))), "fp16 range"),
    (dict(ns=_ns(coefficients=(float("nan"), 0.0, 0.0))), "fp16 range"),
    (dict(ns=_ns(coefficients=(float("inf"), 0.0, 0.0))), "fp16 range"),
    (dict(ns=_ns(coefficients=(3.0, 3.0, 3.0))), "grow"), (dict(ns=_ns(coefficients=(5.0, 0.0, 0.0))), "grow"),
    (dict(ns=_ns(coefficients=(1.9, 0.0, 0.0))), "grow"),  # (only the later steps leave the range)
])
def test_orthogonalize_refuses(kw, message):
    with pytest.raises(_lib.HAError, match=message):
        _orthogonalize(**kw)


def test_orthogonalize_accepts_usual_coefficients_and_nothing_to_do():
    for coefficients in (muon.COEFFICIENTS, (1.5, -0.5, 0.0), (15 / 8, -10 / 8, 3 / 8), (1.0, 0.0, 0.0),
                         [(8.28721, -23.5959, 17.3004), (4.10706, -2.94785, 0.544843), (3.94869, -2.9089, 0.551819),
                          (3.31842, -2.48849, 0.510049), (2.30065, -1.6689, 0.418807)]):
        _orthogonalize(batch=0, ns=_ns(coefficients=coefficients))  # (an empty batch: checked, then nothing runs)
    bad = _ns()
    for steps in (0, 17, -1):
        bad.steps = steps
        with pytest.raises(_lib.HAError, match="steps"):
            _orthogonalize(ns=bad)


def test_muon_step_refuses():
    sc = _lib.MuonScalars(0.95, 0.05, 1, 0, 0, 1.0)

    def call(tab, n=None, rows=64, cols=96, code=_lib.HA_BF16, scalars=sc, peers=None, ws=WS, no_shapes=False):
        shapes = np.asarray([[rows, cols]] * 1, dtype=np.int64)
        _lib.call("ha_muon_step", None if tab is None else _lib.np_ptr(tab), None if no_shapes else _lib.np_ptr(shapes),
                  len(tab) if n is None else n, code,
                  None if scalars is None else ctypes.byref(scalars), ctypes.byref(_ns()), 0,
                  None if peers is None else ctypes.byref(peers), None, None, ws, _bytes(1, 64, 96), None)

    def entry(**kw):
        tab = np.zeros(1, dtype=_lib.TENSOR_DTYPE)
        for name, value in dict(dict(grad=SRC, master=DST, exp_avg=DST + 65536, param=SRC + 65536, numel=64 * 96), **kw).items():
            tab[name] = value
        return tab

    with pytest.raises(_lib.HAError, match="dtype"):
        call(entry(), code=9)
    with pytest.raises(_lib.HAError, match="tensors"):
        call(entry(), n=-1)
    with pytest.raises(_lib.HAError, match="scalars"):
        call(entry(), scalars=None)
    with pytest.raises(_lib.HAError, match="NULL table"):
        call(None, n=1)
    with pytest.raises(_lib.HAError, match="NULL table"):
        call(entry(), no_shapes=True)
    with pytest.raises(_lib.HAError, match="matrices of"):
        call(entry(), rows=0)
    for kw in (dict(numel=64 * 95), dict(master=0), dict(exp_avg=0), dict(param=0)):
        with pytest.raises(_lib.HAError, match="entry 0"):
            call(entry(**kw))
    for kw in (dict(grad=SRC + 1), dict(master=DST + 2), dict(exp_avg=DST + 1), dict(param=SRC + 1)):
        with pytest.raises(_lib.HAError, match="misaligned"):
            call(entry(**kw))
    peers = _lib.Peers()
    peers.n = 1
    peers.delta[0] = 8
    with pytest.raises(_lib.HAError, match="16-byte"):
        call(entry(), peers=peers)
    peers.n = 16
    with pytest.raises(_lib.HAError, match="peers"):
        call(entry(), peers=peers)
    with pytest.raises(_lib.HAError, match="256-byte"):
        call(entry(), ws=WS + 8)
    call(entry(), n=0)  # nothing to do


def test_python_arguments():
    x = torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        orthogonalize(x)
    with pytest.raises(TypeError, match="expected a tensor"):
        orthogonalize([[1.0]])
    with pytest.raises(TypeError, match="dtype"):
        orthogonalize(x.double())
    with pytest.raises(ValueError, match="matrices"):
        orthogonalize(torch.zeros(5))
    for kw, message in ((dict(steps=0), "steps"), (dict(steps=17), "steps"), (dict(coefficients=(1.0, 2.0)), "coefficients"),
                        (dict(coefficients=[(1.5, -0.5, 0.0)] * 4), "coefficients"),
                        (dict(coefficients=[(1.5, -0.5)] * 5), "coefficients"), (dict(coefficients=()), "coefficients")):
        with pytest.raises(ValueError, match=message):
            muon._ns_params(kw.get("steps", 5), kw.get("coefficients", muon.COEFFICIENTS), 1e-7)


def _group(*shapes, **kw):
    return dict({"params": [torch.nn.Parameter(torch.zeros(s)) for s in shapes], "lr": 1e-3}, **kw)


@pytest.mark.parametrize("groups,kw,error,message", [
    ([_group((3, 4))], dict(momentum=1.0), ValueError, "momentum"),
    ([_group((3, 4))], dict(momentum=-0.1), ValueError, "momentum"),
    ([_group((3, 4))], dict(adjust_lr="other"), ValueError, "adjust_lr"),
    ([_group((3, 4))], dict(ns_steps=0), ValueError, "steps"),
    ([_group((3, 4))], dict(ns_coefficients=(1, 2)), ValueError, "coefficients"),
    ([_group((7,), use_muon=True)], {}, ValueError, "two-dimensional"),
    ([_group((2, 3, 4), use_muon=True)], {}, ValueError, "two-dimensional"),
    ([_group((0, 4))], {}, ValueError, "non-empty"),
    ([], {}, ValueError, "ZeroOneMuon received no trainable parameters"),
    ([_group((3, 4))], dict(betas=(0.9, 1.0)), ValueError, "betas"),
    ([_group((3, 4))], {}, RuntimeError, "ZeroOneMuon runs on CUDA devices only"),
    ([_group((0, 4), (5,), use_muon=False)], {}, RuntimeError, "CUDA devices only"),
])
def test_constructor_refuses(groups, kw, error, message):
    with pytest.raises(error, match=message):
        ZeroOneMuon(groups, rank=0, world_size=1, **kw)


def test_layout_keeps_matrices_in_classes_of_their_own():
    numels, codes = [100, 7, 64, 130, 9], [_lib.HA_BF16, _lib.HA_BF16, _lib.HA_F32, _lib.HA_BF16, _lib.HA_F32]
    flags = [True, False, True, True, False]
    for world in (1, 2, 3):
        plain, mixed = layout.plan(numels, codes, world), layout.plan(numels, codes, world, flags)
        assert mixed.owner == plain.owner  # ownership goes by size alone
        assert [(c.code, c.muon, c.indices) for c in mixed.classes] == [
            (_lib.HA_F32, False, [4]), (_lib.HA_F32, True, [2]), (_lib.HA_BF16, False, [1]), (_lib.HA_BF16, True, [0, 3])]
        assert [(c.code, c.muon, c.indices) for c in plain.classes] == [
            (_lib.HA_F32, False, [2, 4]), (_lib.HA_BF16, False, [0, 1, 3])]
        for c in mixed.classes:  # slots of a class do not overlap within an owner's segment
            for r in range(world):
                slots = sorted((c.offset[i], numels[i]) for i in c.owned(mixed.owner, r))
                for (a, n), (b, _) in zip(slots, slots[1:]):
                    assert a + n <= b
