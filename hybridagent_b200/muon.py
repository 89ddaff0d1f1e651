"""Muon: orthogonalised momentum updates for the matrices of a model, with ZeRO-1 sharding.

``orthogonalize(x)`` replaces each matrix by one with the same singular vectors and singular values
pushed towards 1, by Newton-Schulz steps ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` (five
steps with K. Jordan's coefficients by default, which leave them between about 0.7 and 1.2).

``ZeroOneMuon`` is ``ZeroOneAdamW`` with that update for matrices: the same construction,
``zero_grad`` / ``all_reduce_grads`` / ``clip_grad_norm`` / ``step``, ownership, exchange, checkpoints
and changed-group writes.  A tensor is owned whole by one rank, so its momentum and the products on
it stay on one GPU; per matrix with gradient g:

    M <- mu M + (1 - mu) g;   U = (1 - mu) g + mu M  (nesterov) or M
    W <- W (1 - lr weight_decay) - lr f orthogonalize(U)

with f from ``adjust_lr``: "match_rms_adamw" 0.2 sqrt(max(rows, cols)), which gives the update AdamW's
usual size so that its learning rates carry over, "original" sqrt(max(1, rows / cols)), or None for 1.
Momentum and masters are fp32.  The reference trains every tensor with AdamW
(hybrid_rl/optimizer.py:162-194); it has no counterpart of this class.

The products run on fp16 operands with fp32 accumulators in ``libhybridagent_b200.so``
(``ha_orthogonalize``, ``ha_muon_step``).  Five steps with the default coefficients, as bf16, are within
2.3e-3 (relative, 2-norm) of the exact iteration where singular values are alike or fall off slowly, and within 6e-3 where
most of them vanish (a gradient of few samples); rounding to bf16 alone is 1.7e-3.  Further steps bring up what
rounding leaves in directions that a matrix does not have, 3.44-fold each: matrices of rank 4 are off by up to 5e-3 after
six steps, 1e-2 after eight and 1e-1 after ten (2e-2 with fp32 products).
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator
import os

import numpy as np
import torch

from . import _lib
from .optimizer import _CODES, ZeroOneAdamW

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
ADJUST_LR = ("match_rms_adamw", "original", None)


def _ns_params(steps: int, coefficients, eps: float) -> _lib.NsParams:
    """``coefficients``: one (a, b, c) for every step, or one for each."""
    steps = operator.index(steps)
    if not 1 <= steps <= _lib.HA_NS_MAX_STEPS:
        raise ValueError(f"steps must be between 1 and {_lib.HA_NS_MAX_STEPS}")
    coefficients = list(coefficients)
    each = bool(coefficients) and hasattr(coefficients[0], "__len__")
    rows = [tuple(float(v) for v in row) for row in (coefficients if each else [coefficients] * steps)]
    if len(rows) != steps or any(len(row) != 3 for row in rows):
        raise ValueError("coefficients must be (a, b, c), or one (a, b, c) for each step")
    out = _lib.NsParams()
    out.steps = steps
    out.eps = float(eps)
    out.coef[:3 * steps] = [v for row in rows for v in row]
    return out


@functools.lru_cache(maxsize=64)
def _usual_params(steps: int, eps: float) -> _lib.NsParams:
    return _ns_params(steps, COEFFICIENTS, eps)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(batch: int, rows: int, cols: int) -> int:
    out = ctypes.c_size_t(0)
    _lib.call("ha_orthogonalize_workspace", batch, rows, cols, ctypes.byref(out))
    return out.value


def _budget(name: str, default: int) -> int:
    value = int(os.environ.get(name, str(default)))
    if value < 0:
        raise ValueError(f"{name}={value}: expected >= 0")
    return value


def _workspace(size: int, least: int, device: torch.device) -> torch.Tensor:
    """`size` bytes on `device`, or half of it, a quarter, ... but `least`, where memory is short."""
    while True:
        try:
            return torch.empty(size, dtype=torch.uint8, device=device)
        except torch.OutOfMemoryError:
            if size <= least:
                raise
            size = max(size // 2, least)


def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The Newton-Schulz orthogonalisation of ``x`` (..., rows, cols), each matrix for itself, as bf16.

    ``x`` is fp32, bf16 or fp16 on a CUDA device; matrices that are not contiguous are copied first, but for
    transposed views of contiguous ones, whose result is such a view too unless ``out`` is given.
    ``out`` (bf16, contiguous, of x's shape, not overlapping it) receives the result if given.  A matrix
    is divided by its Frobenius norm, or by ``eps`` where that is larger, so a zero matrix stays zero.
    One with a non-finite element becomes NaN.  Not differentiable.  Runs on the current stream of x's
    device without waiting for it and may be captured into a CUDA graph; temporary memory of up to
    HYBRIDAGENT_B200_NS_BYTES (default 8 GiB; at least one matrix's planes) comes from torch, less where that much is
    not free."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"expected a tensor, got {type(x).__name__}")
    if x.dtype not in _CODES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if x.ndim < 2:
        raise ValueError(f"expected matrices (..., rows, cols), got shape {tuple(x.shape)}")
    if x.device.type != "cuda":
        raise RuntimeError(f"orthogonalize runs on CUDA devices only; the tensor is on {x.device} "
                           "(there is no CPU path)")
    if coefficients is COEFFICIENTS and type(steps) is int and type(eps) is float:
        ns = _usual_params(steps, eps)
    else:
        ns = _ns_params(steps, coefficients, eps)
    if x.requires_grad:
        x = x.detach()
    if out is not None:
        if out.dtype != torch.bfloat16 or out.shape != x.shape or out.device != x.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous bfloat16 tensor of shape {tuple(x.shape)} on {x.device}")
    elif x.mT.is_contiguous() and not x.is_contiguous():  # a transposed view: its transpose lies in order
        return orthogonalize(x.mT, steps=steps, coefficients=coefficients, eps=eps).mT
    rows, cols = x.shape[-2:]
    src = x.contiguous()
    given = out is not None
    if not given:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    elif src is x and _overlap(x, out):
        raise ValueError("out overlaps x")
    if src.numel() == 0:
        return out
    batch = src.numel() // (rows * cols)
    size, least = _workspace_bytes(batch, rows, cols), _workspace_bytes(1, rows, cols)
    budget = _budget("HYBRIDAGENT_B200_NS_BYTES", 8 << 30)
    if size > budget:
        size = max(budget, least)
    ws = _workspace(size, least, x.device)
    device = x.device.index
    args = ("ha_orthogonalize", src.data_ptr(), _CODES[x.dtype], out.data_ptr(), batch, rows, cols, ctypes.byref(ns),
            ws.data_ptr(), ws.numel(), torch._C._cuda_getCurrentRawStream(device))
    if device == torch._C._cuda_getDevice():
        _lib.call(*args)
    else:
        with torch.cuda.device(device):
            _lib.call(*args)
    if given:
        torch.autograd.graph.increment_version(out)  # written through its address
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    a0, b0 = a.data_ptr(), b.data_ptr()
    return a0 < b0 + b.numel() * b.element_size() and b0 < a0 + a.numel() * a.element_size()


class ZeroOneMuon(ZeroOneAdamW):
    """ZeRO-1 Muon for matrices and AdamW for the rest (see the module's docstring).

    A group's ``"use_muon"`` says which update its tensors take; without it two-dimensional tensors
    take Muon's and all others AdamW's.  Embeddings and output heads are usually given
    ``"use_muon": False``.  ``betas`` and ``eps`` belong to the AdamW tensors, ``weight_decay`` to both.
    ``exp_avg`` holds a Muon tensor's momentum; it has no ``exp_avg_sq``.  Workspace for the products, of
    HYBRIDAGENT_B200_MUON_BYTES (default 4 GiB, at least the largest owned matrix's need and no more than
    all of them need; less where that much is not free), is held for the optimizer's life."""

    state_format = "hybridagent_b200.zero1_muon/1"
    _updates = ("AdamW", "Muon")

    def __init__(self, param_groups, *, rank: int, world_size: int, momentum: float = 0.95, nesterov: bool = True,
                 ns_steps: int = 5, ns_coefficients=COEFFICIENTS, ns_eps: float = 1e-7,
                 adjust_lr: str | None = "match_rms_adamw", betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, comm_timeout_s: float | None = None, land_grads: bool = False):
        self.momentum = float(momentum)
        self.nesterov = bool(nesterov)
        self.adjust_lr = adjust_lr
        if not 0.0 <= self.momentum < 1.0:
            raise ValueError("momentum must be in [0, 1)")
        if adjust_lr not in ADJUST_LR:
            raise ValueError(f"adjust_lr must be one of {ADJUST_LR}, got {adjust_lr!r}")
        self._ns = _ns_params(ns_steps, ns_coefficients, ns_eps)
        super().__init__(param_groups, rank=rank, world_size=world_size, betas=betas, eps=eps,
                         weight_decay=weight_decay, comm_timeout_s=comm_timeout_s, land_grads=land_grads)
        muon = [c for c in self._classes if c.muon and c.owned]
        with torch.cuda.device(self.device):
            size, least, budget = 0, 0, _budget("HYBRIDAGENT_B200_MUON_BYTES", 4 << 30)
            for c in muon:
                shapes = [tuple(self.params[i].shape) for i in c.owned]
                # equal shapes follow one another: they run together
                c.order = np.asarray(sorted(range(len(shapes)), key=lambda k: shapes[k]), dtype=np.int64)
                c.shapes = np.ascontiguousarray([shapes[k] for k in c.order], dtype=np.int64)
                need = sum(_workspace_bytes(1, *s) for s in shapes)
                least = max(least, *(_workspace_bytes(1, *s) for s in set(shapes)), 0)
                size = max(size, min(need, max(budget, least)))
                c.neg_lr = np.asarray([-(self.lrs[i] * self._factor(*self.params[i].shape)) for i in c.owned],
                                      dtype=np.float32)
            self._muon_ws = _workspace(size, least, self.device) if size else None
            # set by a step whose products gave up; pinned host memory, which the GPU writes itself
            self._muon_status = torch.zeros(1, dtype=torch.int32, pin_memory=True)
            torch.cuda.current_stream().synchronize()

    def _takes_muon(self, parameter: torch.Tensor, group: dict) -> bool:
        wanted = group.get("use_muon", parameter.ndim == 2)
        if wanted and parameter.ndim != 2:
            raise ValueError(f"use_muon needs two-dimensional parameters, got shape {tuple(parameter.shape)}")
        if wanted and parameter.numel() == 0:
            raise ValueError(f"use_muon needs non-empty matrices, got shape {tuple(parameter.shape)}")
        return bool(wanted)

    def _factor(self, rows: int, cols: int) -> float:
        if self.adjust_lr == "match_rms_adamw":
            return 0.2 * math.sqrt(max(rows, cols))
        if self.adjust_lr == "original":
            return math.sqrt(max(1.0, rows / cols))
        return 1.0

    def _update_muon(self, c, sc: _lib.AdamwScalars, changed_only: bool, p2p: bool) -> None:
        """The Muon update of class c's owned matrices that have a gradient."""
        ms = _lib.MuonScalars(np.float32(self.momentum), np.float32(1.0 - self.momentum), int(self.nesterov),
                              sc.use_decay, sc.clip, sc.clip_mult)
        table = np.ascontiguousarray(c.table.np[c.order])
        _lib.call("ha_muon_step", _lib.np_ptr(table), _lib.np_ptr(c.shapes), len(table), c.code, ctypes.byref(ms),
                  ctypes.byref(self._ns), int(changed_only), ctypes.byref(c.peers) if p2p else None,
                  c.changed_dev.data_ptr() if changed_only else None, self._muon_status.data_ptr(),
                  self._muon_ws.data_ptr(), self._muon_ws.numel(), self._stream())
        # momentum, load and weights, and one run of the products: more where the workspace or a launch's
        # parameters split them
        self.launches += 4

    def _check_status(self) -> None:
        """Raises if the products of a step that has run gave up."""
        if int(self._muon_status[0]) != 0:
            raise RuntimeError("Muon step: a wait inside the Newton-Schulz products of an earlier step ran out.  Matrices of "
                               "that step kept their weights (all but those of passes through the workspace that were "
                               "done before), while momenta, step counts and other tensors advanced: load a checkpoint "
                               "(load_state_dict) to go on")

    def step(self) -> None:
        """``ZeroOneAdamW.step`` with Muon's update of the matrices.  Raises, before anything changes, if the products of an
        earlier step are known to have given up."""
        self._check_status()
        super().step()

    def state_dict(self) -> dict:
        state = super().state_dict()  # (waits for the steps before)
        self._check_status()
        return state

    def load_state_dict(self, state: dict) -> None:
        super().load_state_dict(state)  # (waits for the steps before)
        self._muon_status.zero_()

    def state_summary(self) -> str:
        n = sum(len(c.layout.indices) for c in self._classes if c.muon)
        return (f"ZeRO-1 FP32 Muon: {n} matrices, AdamW: {len(self.params) - n} tensors; rank {self.rank} owns "
                f"{self.owned_numel / 1e6:.1f}M parameters")
