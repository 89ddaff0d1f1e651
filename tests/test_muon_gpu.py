"""Newton-Schulz orthogonalisation and the Muon step against their definitions in 64 bits.

Tolerances (2-norm, relative).  Every stored fp16 value is off by at most half a step, 2^-11.  A step
stores A, its factor and X; taking its three roundings, in each of five steps, as independent and of
their full size, with 3.45, the most that a step multiplies by, as the weight of each, gives
sqrt(15) * 3.45 * 2^-11 = 6.5e-3.  A result stored as bf16 adds half a step of its own, 2^-8."""
import ctypes
import math

import numpy as np
import pytest

from helpers import to_torch
from hybridagent_b200 import _lib, muon

pytestmark = pytest.mark.gpu

NS = math.sqrt(15) * 3.45 * 2.0 ** -11
NS_BF16 = NS + 2.0 ** -8


def definition(x, steps=5, coefficients=muon.COEFFICIENTS, eps=1e-7):
    """The steps in 64 bits on the matrices of x (..., rows, cols)."""
    x = x.double()
    if x.shape[-2] > x.shape[-1]:
        return definition(x.mT, steps, coefficients, eps).mT
    rows = coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    for a, b, c in rows:
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def off(got, want):
    """Largest relative error of a matrix."""
    d = (got.double() - want).square().sum((-2, -1)).sqrt()
    return float((d / want.square().sum((-2, -1)).sqrt()).max())


def values(kind, shape, dtype, seed=0, scale=1e-4):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda")
    if kind == "graded":  # a few strong directions over weak noise
        k = min(4, *shape[-2:])
        x = 0.05 * x + (torch.randn(*shape[:-1], k, generator=gen, device="cuda") @
                        torch.randn(*shape[:-2], k, shape[-1], generator=gen, device="cuda"))
    return (x * scale).to(dtype)


SHAPES = [(1, 1, 1), (1, 1, 40), (2, 37, 1), (1, 2, 3), (3, 16, 16), (1, 31, 33), (2, 64, 64), (1, 64, 96), (2, 96, 64),
          (1, 127, 129), (1, 128, 128), (2, 128, 1000), (1, 129, 127), (2, 5, 2047), (1, 2047, 6), (3, 100, 4097),
          (1, 4097, 120), (2, 200, 333), (2, 333, 200), (1, 255, 257), (1, 256, 256), (2, 256, 512), (3, 512, 256),
          (1, 257, 641), (1, 513, 512), (2, 700, 1500), (1, 1500, 700), (5, 640, 1280), (1, 1000, 1537), (1, 1024, 4096),
          (1, 4096, 1024), (1, 2300, 2177)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize(shape, dtype):
    import torch
    from hybridagent_b200 import orthogonalize
    # (fp16 gradients are scaled up, as training with them does)
    x = values("normal", shape, getattr(torch, dtype), scale=1e-4 if dtype != "float16" else 1e-1)
    y = orthogonalize(x)
    assert y.shape == x.shape and y.dtype == torch.bfloat16 and y.is_contiguous()
    assert off(y, definition(x)) <= NS_BF16


@pytest.mark.parametrize("shape", [(2, 24, 300), (1, 64, 64), (1, 120, 2500), (1, 2500, 100), (2, 256, 512), (1, 900, 700),
                                   (1, 704, 2816), (1, 3000, 800)], ids=lambda s: "x".join(map(str, s)))
def test_graded_spectrum(shape):
    import torch
    from hybridagent_b200 import orthogonalize
    x = values("graded", shape, torch.float32, seed=3)
    assert off(orthogonalize(x), definition(x)) <= NS_BF16


@pytest.mark.parametrize("steps,coefficients", [(1, muon.COEFFICIENTS), (2, muon.COEFFICIENTS), (3, muon.COEFFICIENTS),
                                                (4, muon.COEFFICIENTS), (5, (1.5, -0.5, 0.0)), (6, (15 / 8, -10 / 8, 3 / 8)),
                                                (16, (1.5, -0.5, 0.0)),
                                                (5, [(8.28721, -23.5959, 17.3004), (4.10706, -2.94785, 0.544843),
                                                     (3.94869, -2.9089, 0.551819), (3.31842, -2.48849, 0.510049),
                                                     (2.30065, -1.6689, 0.418807)])])
@pytest.mark.parametrize("shape", [(2, 60, 80), (1, 300, 500), (1, 1400, 660)], ids=lambda s: "x".join(map(str, s)))
def test_other_steps_and_coefficients(shape, steps, coefficients):
    import torch
    from hybridagent_b200 import orthogonalize
    x = values("normal", shape, torch.float32, seed=steps)
    rows = coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    # the module's bound with this schedule's own factors: a step multiplies by at most its a
    bound = math.sqrt(3 * steps) * max(max(abs(r[0]) for r in rows), 1.0) * 2.0 ** -11 + 2.0 ** -8
    want = definition(x, steps, coefficients)
    assert off(orthogonalize(x, steps=steps, coefficients=coefficients), want) <= bound


@pytest.mark.parametrize("shape", [(40, 60), (300, 200), (700, 1500)], ids=lambda s: "x".join(map(str, s)))
def test_zero_and_nonfinite_matrices_stay_to_themselves(shape):
    import torch
    from hybridagent_b200 import orthogonalize
    x = values("normal", (6, *shape), torch.float32, seed=1)
    clean = orthogonalize(x)
    x[1] = 0
    x[2, shape[0] // 2, 3] = math.inf
    x[3, 0, shape[1] - 1] = -math.inf
    x[4, shape[0] - 1, 0] = math.nan
    y = orthogonalize(x)
    assert (y[1] == 0).all()
    for k in (2, 3, 4):
        assert y[k].isnan().all()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[5], clean[5])


def test_scale_does_not_matter_until_eps():
    import torch
    from hybridagent_b200 import orthogonalize
    for shape in ((50, 70), (260, 520)):
        x = values("normal", shape, torch.float32, scale=1.0)
        y = orthogonalize(x, eps=1e-30)
        for k in (-80, -30, 30, 80):  # powers of two: the same bits after the division
            assert torch.equal(orthogonalize(x * 2.0 ** k, eps=1e-30), y)
        # below eps the matrix is divided by eps: small, and amplified by a in every step
        tiny = x / x.norm() * 1e-4
        got, want = orthogonalize(tiny, eps=1.0).double(), definition(tiny, eps=1.0)
        assert float((got - want).norm() / want.norm()) <= NS_BF16


def test_layouts_out_and_streams():
    import torch
    from hybridagent_b200 import orthogonalize
    base = values("normal", (3, 2, 90, 128), torch.bfloat16, seed=5)
    want = orthogonalize(base)
    assert off(want, definition(base)) <= NS_BF16
    assert torch.equal(orthogonalize(base.mT).mT, want)                        # transposed views
    wide = torch.zeros(3, 2, 90, 200, dtype=torch.bfloat16, device="cuda")
    wide[..., 7:135] = base
    assert torch.equal(orthogonalize(wide[..., 7:135]), want)                  # row stride and odd start
    assert torch.equal(orthogonalize(base[:, 1]), want[:, 1])                  # batch stride
    flat = torch.zeros(base.numel() + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = base.reshape(-1)
    assert torch.equal(orthogonalize(flat[1:].view(base.shape)), want)         # aligned to an element only
    out = torch.full((base.numel() + 9,), 7.0, dtype=torch.bfloat16, device="cuda")
    got = orthogonalize(base, out=out[1:-8].view(base.shape))                  # odd start of the result
    assert got.data_ptr() == out[1:].data_ptr() and torch.equal(got, want)
    assert float(out[0]) == 7.0 and (out[-8:] == 7.0).all()                    # nothing else is written
    with pytest.raises(ValueError, match="overlap"):
        orthogonalize(base, out=base)
    for bad in (torch.empty(3, 2, 90, 127, dtype=torch.bfloat16, device="cuda"),
                torch.empty(base.shape, dtype=torch.float16, device="cuda"), torch.empty(base.shape, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="out must be"):
            orthogonalize(base, out=bad)
    for empty in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        assert orthogonalize(torch.empty(empty, device="cuda")).shape == torch.Size(empty)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = []
    for k in range(4):  # two calls at once, on two streams
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            results.append(orthogonalize(base))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)
    p = torch.nn.Parameter(base.clone())
    assert not orthogonalize(p).requires_grad


@pytest.mark.parametrize("shape", [(4, 64, 96), (2, 300, 700)], ids=lambda s: "x".join(map(str, s)))
def test_captured_graphs_replay_with_new_values(shape):
    import torch
    from hybridagent_b200 import orthogonalize
    xs = [values("normal", shape, torch.float32, seed=k) for k in range(3)]
    static = [x.clone() for x in xs[:2]]
    orthogonalize(static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:  # two graphs, each with the memory that its capture took
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(orthogonalize(s))
        graphs.append(g)
    for rep in range(2):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, o in zip(static, outs):
            assert torch.equal(o, orthogonalize(s))
        for s in static:
            s.copy_(xs[2])


def test_workspace_budget_splits_the_batch(monkeypatch):
    import torch
    from hybridagent_b200 import orthogonalize
    x = values("normal", (7, 150, 260), torch.bfloat16, seed=9)
    want = orthogonalize(x)
    one = muon._workspace_bytes(1, 150, 260)
    for budget in (0, 2 * one, 3 * one + 12345):
        monkeypatch.setenv("HYBRIDAGENT_B200_NS_BYTES", str(budget))
        assert off(orthogonalize(x), definition(x)) <= NS_BF16
        assert float((orthogonalize(x).float() - want.float()).abs().max()) <= 2.0 ** -8
    monkeypatch.setenv("HYBRIDAGENT_B200_NS_BYTES", "-1")
    with pytest.raises(ValueError, match="NS_BYTES"):
        orthogonalize(x)


def test_offsets_beyond_32_bits(monkeypatch):
    import torch
    from hybridagent_b200 import orthogonalize
    monkeypatch.setenv("HYBRIDAGENT_B200_NS_BYTES", str(40 << 30))  # all in one pass
    n = 1100  # x 704 x 2816: 2.18e9 elements
    assert n * 704 * 2816 > 2 ** 31
    x = torch.empty(n, 704, 2816, dtype=torch.bfloat16, device="cuda")
    for k in range(0, n, 100):
        x[k:k + 100] = values("normal", (100, 704, 2816), torch.bfloat16, seed=k)
    y = orthogonalize(x)
    for k in (0, 541, 1083, 1099):
        assert off(y[k], definition(x[k])) <= NS_BF16


# ---------------------------------------------------------------- the optimizer
SETS = {
    "small": ([(64, 96), (96, 64), (33, 70), (33, 70), (128, 300), (1, 50)], [(1000,), (7,), (3, 5, 2)]),
    "medium": ([(256, 512), (256, 512), (512, 256), (700, 300), (641, 1300)], [(4099,)]),
}


def build(kind, dtype, seed=0, lr=2e-2, **kw):
    import torch
    from hybridagent_b200 import ZeroOneMuon
    mats, rest = SETS[kind]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    params = [torch.nn.Parameter((torch.randn(s, generator=gen, device="cuda") * 0.02).to(dtype)) for s in mats + rest]
    opt = ZeroOneMuon([{"params": params[:len(mats)], "lr": lr}, {"params": params[len(mats):], "lr": 1e-3}], rank=0,
                      world_size=1, weight_decay=0.01, **kw)
    return params, opt, len(mats)


def set_grads(params, step, dtype, skip=()):
    for i, p in enumerate(params):
        p.grad = None if i in skip else values("normal", p.shape, dtype, seed=100 * step + i, scale=0.05)


class Definition:
    """The Muon tensors' update in 64 bits, from the optimizer's state at construction."""

    def __init__(self, opt, n, factor, momentum=0.95, nesterov=True, lr=2e-2, decay=0.01):
        self.w = [opt.master[i].double().clone() for i in range(n)]
        self.m = [w.new_zeros(w.shape) for w in self.w]
        self.moved = [0.0] * n
        self.factor, self.mu, self.nesterov, self.lr, self.decay = factor, momentum, nesterov, lr, decay

    def step(self, i, p, scale):
        g = p.grad.double()
        if scale is not None:  # the clip is applied in the gradient's type, as grad.mul_ does
            g = (p.grad.float() * np.float32(scale)).to(p.dtype).double()
        self.m[i] = self.mu * self.m[i] + (1 - self.mu) * g
        u = (1 - self.mu) * g + self.mu * self.m[i] if self.nesterov else self.m[i]
        d = self.lr * self.factor(*p.shape) * definition(u)
        self.w[i] = self.w[i] * (1 - self.lr * self.decay) - d
        self.moved[i] += float(d.norm())

    def check(self, i, opt, p, steps):
        import torch
        # momentum: fp32, two roundings in each step
        err = float((opt.exp_avg[i].double() - self.m[i]).norm() / self.m[i].norm())
        assert err <= 2 * steps * 2.0 ** -24, f"momentum[{i}]: {err}"
        # masters: the products' error on what moved, and two roundings of the weight in each step
        err = float((opt.master[i].double() - self.w[i]).norm())
        assert err <= NS * self.moved[i] + 2 * steps * 2.0 ** -24 * float(self.w[i].norm()), f"master[{i}]: {err}"
        assert torch.equal(p.data, opt.master[i].to(p.dtype)), f"param[{i}] is not its rounded master"


FACTORS = {"match_rms_adamw": lambda r, c: 0.2 * math.sqrt(max(r, c)), "original": lambda r, c: math.sqrt(max(1, r / c)),
           None: lambda r, c: 1.0}


@pytest.mark.parametrize("kind", list(SETS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("kw", [dict(), dict(adjust_lr="original", nesterov=False, momentum=0.8), dict(adjust_lr=None, momentum=0.0)],
                         ids=["default", "original_plain", "none_no_momentum"])
def test_optimizer_steps(kind, dtype, kw):
    """Several steps in the trainer's order: clipped and unclipped, one without some gradients."""
    import torch
    dt = getattr(torch, dtype)
    params, opt, n = build(kind, dt, **kw)
    ref = Definition(opt, n, FACTORS[kw.get("adjust_lr", "match_rms_adamw")], kw.get("momentum", 0.95),
                     kw.get("nesterov", True))
    done = [0] * n
    for step, (max_norm, skip) in enumerate([(1.0, ()), (1e9, ()), (0.5, (1, 3)), (0.0, ())]):
        opt.zero_grad(set_to_none=True)
        set_grads(params, step, dt, skip)
        opt.all_reduce_grads()
        norm = opt.clip_grad_norm(max_norm)
        scale = max_norm / (norm + 1e-6) if max_norm > 0 and norm > max_norm else None
        for i in range(n):
            if i not in skip:
                ref.step(i, params[i], scale)
                done[i] += 1
        opt.step()
    for i in range(n):
        assert opt.param_steps[i] == done[i]
        assert i not in opt.exp_avg_sq
        ref.check(i, opt, params[i], done[i])
    assert opt.step_count == 4


def test_other_tensors_take_adamw_bit_for_bit():
    import torch
    from hybridagent_b200 import ZeroOneAdamW, ZeroOneMuon
    shapes = [(50, 60), (1000,), (7,), (33, 44)]
    def make(cls, **flags):
        gen = torch.Generator(device="cuda").manual_seed(2)
        ps = [torch.nn.Parameter((torch.randn(s, generator=gen, device="cuda") * 0.02).bfloat16()) for s in shapes]
        return ps, cls([{"params": ps, "lr": 1e-3, **flags}], rank=0, world_size=1, weight_decay=0.01)
    a_params, a = make(ZeroOneAdamW)
    b_params, b = make(ZeroOneMuon, use_muon=False)
    for step in range(3):
        for ps, opt in ((a_params, a), (b_params, b)):
            set_grads(ps, step, torch.bfloat16)
            opt.all_reduce_grads()
            opt.clip_grad_norm(1.0)
            opt.step()
    for i in range(len(shapes)):
        assert torch.equal(a_params[i].data, b_params[i].data)
        for name in ("master", "exp_avg", "exp_avg_sq"):
            assert torch.equal(getattr(a, name)[i], getattr(b, name)[i])


def test_changed_sector_writes_and_writes_behind_the_optimizer():
    import torch
    params, opt, n = build("medium", torch.bfloat16, lr=1e-6)
    modes = []
    for step in range(4):
        if step == 2:
            with torch.no_grad():
                params[1].mul_(1.5)  # overwritten with the rounded master by the next step
        set_grads(params, step, torch.bfloat16)
        opt.clip_grad_norm(1.0)
        opt.step()
        modes.append(opt.write_stats()["mode"])
        for i in range(n):
            assert torch.equal(params[i].data, opt.master[i].bfloat16())
    assert modes == ["changed groups", "changed groups", "full", "changed groups"]
    stats = opt.write_stats()
    assert 0 < stats["changed_groups"] < stats["groups"] // 2


def test_state_dict_and_checkpoints(tmp_path):
    import torch
    from hybridagent_b200 import ZeroOneAdamW, ZeroOneMuon, checkpoint
    params, opt, n = build("small", torch.bfloat16)
    for step in range(2):
        set_grads(params, step, torch.bfloat16)
        opt.clip_grad_norm(1.0)
        opt.step()
    checkpoint.save_optimizer_state(opt, tmp_path)
    fresh = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = ZeroOneMuon([{"params": fresh[:n], "lr": 2e-2}, {"params": fresh[n:], "lr": 1e-3}], rank=0, world_size=1,
                        weight_decay=0.01)
    checkpoint.load_optimizer_state(again, tmp_path)
    assert again.step_count == 2
    for ps, o in ((params, opt), (fresh, again)):
        set_grads(ps, 7, torch.bfloat16)
        o.clip_grad_norm(1.0)
        o.step()
    for i in range(len(params)):
        assert torch.equal(params[i].data, fresh[i].data)
        assert torch.equal(opt.master[i], again.master[i]) and torch.equal(opt.exp_avg[i], again.exp_avg[i])
    adamw = ZeroOneAdamW([{"params": [torch.nn.Parameter(p.detach().clone()) for p in params], "lr": 1e-3}], rank=0,
                         world_size=1)
    with pytest.raises(ValueError, match="state dict"):
        adamw.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="state dict"):
        opt.load_state_dict(adamw.state_dict())
    assert "6 matrices" in opt.state_summary()


def test_steps_and_landing_are_deterministic():
    """The same steps twice, and with the norm taken while gradients land: the same bits."""
    import torch
    results = []
    for kw in ({}, {}, {"land_grads": True}):
        params, opt, n = build("medium", torch.bfloat16, **kw)
        for step in range(2):
            opt.zero_grad(set_to_none=True)
            grads = [values("normal", p.shape, torch.bfloat16, seed=step * 50 + i, scale=0.05) for i, p in enumerate(params)]
            sum((p * g).sum(dtype=torch.float32) for p, g in zip(params, grads)).backward()
            opt.all_reduce_grads()
            opt.clip_grad_norm(1.0)
            opt.step()
        if kw:
            assert opt.land_norm_steps == 2
        results.append([opt.master[i].clone() for i in range(len(params))] + [p.data.clone() for p in params])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_step_through_a_small_workspace_and_many_tensors(monkeypatch):
    """More matrices than a launch's parameters hold, in a workspace that holds a few."""
    import torch
    from hybridagent_b200 import ZeroOneMuon
    shape, count = (20, 30), 130
    def run(budget):
        monkeypatch.setenv("HYBRIDAGENT_B200_MUON_BYTES", str(budget))
        params = [torch.nn.Parameter(values("normal", shape, torch.float32, seed=i, scale=0.02)) for i in range(count)]
        opt = ZeroOneMuon([{"params": params, "lr": 1e-2}], rank=0, world_size=1)
        set_grads(params, 3, torch.float32, skip=(5, 77))
        opt.clip_grad_norm(1.0)
        opt.step()
        return params, opt
    a, opt = run(1 << 30)
    b, _ = run(9 * muon._workspace_bytes(1, *shape))
    for i, (x, y) in enumerate(zip(a, b)):
        start = values("normal", shape, torch.float32, seed=i, scale=0.02)
        if i in (5, 77):
            assert torch.equal(x, start) and torch.equal(y, start)
        else:
            moved = float((x - start).detach().norm())
            assert moved > 0 and float((x - y).detach().norm()) <= 2 * NS * moved


@pytest.mark.parametrize("code,changed_only", [(0, 0), (1, 0), (1, 1), (2, 1)])
def test_muon_step_writes_the_peers_copies(code, changed_only):
    """Peer copies, emulated by a second buffer on this GPU: new values at the same offsets, and with
    changed_only only the stored sectors."""
    import torch
    dt = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}[code]
    rows, cols, n = 48, 72, 3
    numel = rows * cols
    master = [values("normal", (rows, cols), torch.float32, seed=k, scale=0.02) for k in range(n)]
    params = torch.zeros(2, n * numel, dtype=dt, device="cuda")
    if code == 0:
        for k in range(n):
            params[0, k * numel:(k + 1) * numel] = master[k].reshape(-1)
    else:
        for k in range(n):
            params[:, k * numel:(k + 1) * numel] = master[k].reshape(-1).to(dt)
    sentinel = params[1].clone()
    grads = [values("normal", (rows, cols), dt, seed=20 + k, scale=0.1) for k in range(n)]
    mom = [torch.zeros(rows, cols, device="cuda") for _ in range(n)]
    tab = np.zeros(n, dtype=_lib.TENSOR_DTYPE)
    for k in range(n):
        tab[k]["grad"] = grads[k].data_ptr()
        here = params[0, k * numel:].data_ptr()
        tab[k]["master"] = here if code == 0 else master[k].data_ptr()
        tab[k]["param"] = 0 if code == 0 else here
        tab[k]["exp_avg"] = mom[k].data_ptr()
        tab[k]["numel"] = numel
        tab[k]["decay"] = 1.0
        tab[k]["neg_lr"] = -1e-7 if k == 1 else -1e-2
    peers = _lib.Peers()
    peers.n = 1
    peers.delta[0] = params[1].data_ptr() - params[0].data_ptr()
    assert peers.delta[0] % 16 == 0
    before = params.clone()
    ns = muon._ns_params(5, muon.COEFFICIENTS, 1e-7)
    sc = _lib.MuonScalars(0.95, 0.05, 1, 0, 0, 1.0)
    ws = torch.empty(muon._workspace_bytes(n, rows, cols), dtype=torch.uint8, device="cuda")
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    shapes = np.asarray([[rows, cols]] * n, dtype=np.int64)
    _lib.call("ha_muon_step", _lib.np_ptr(tab), _lib.np_ptr(shapes), n, code, ctypes.byref(sc), ctypes.byref(ns), changed_only,
              ctypes.byref(peers), count.data_ptr(), status.data_ptr(), ws.data_ptr(), ws.numel(),
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert int(status) == 0
    if code:
        for k in range(n):
            assert torch.equal(params[0, k * numel:(k + 1) * numel].view(rows, cols), master[k].to(dt))
    assert torch.equal(params[0], params[1])
    moved = (params[0] != before[0]).view(n, numel).sum(1)
    assert int(moved[0]) > numel // 2 and int(moved[2]) > numel // 2
    if changed_only:
        groups = int(count)
        assert int((params[0] != before[0]).view(-1, 16).any(1).sum()) * 4 == groups < 3 * numel // 4
    else:
        assert int(count) == 0
    assert code == 0 or int(moved[1]) < numel // 4  # a step of 1e-7 leaves most rounded values
    assert sentinel.numel() == params[1].numel()


def test_training_loop():
    """A small network in the trainer's order: gradients agree with differences of the loss, and every
    step moves the weights by the definition's update of those gradients."""
    import torch
    from hybridagent_b200 import ZeroOneMuon
    torch.manual_seed(4)
    model = torch.nn.Sequential(torch.nn.Linear(40, 64), torch.nn.GELU(), torch.nn.Linear(64, 24)).cuda()
    x, y = torch.randn(32, 40, device="cuda"), torch.randn(32, 24, device="cuda")
    params = list(model.parameters())
    opt = ZeroOneMuon([{"params": params, "lr": 1e-2}], rank=0, world_size=1)
    mats = [i for i, p in enumerate(params) if p.ndim == 2]
    assert all(i not in opt.exp_avg_sq for i in mats) and len(opt.exp_avg_sq) == 2
    def loss():
        return torch.nn.functional.mse_loss(model(x), y)
    for step in range(3):
        opt.zero_grad(set_to_none=True)
        loss().backward()
        if step == 0:  # central differences in 64 bits along one direction
            import copy
            m64 = copy.deepcopy(model).double()
            d = [torch.randn_like(p, dtype=torch.float64) for p in m64.parameters()]
            def at(h):
                with torch.no_grad():
                    for p, q, v in zip(m64.parameters(), params, d):
                        p.copy_(q.double() + h * v)
                    return float(torch.nn.functional.mse_loss(m64(x.double()), y.double()))
            slope = (at(1e-5) - at(-1e-5)) / 2e-5
            dot = sum(float((p.grad.double() * v).sum()) for p, v in zip(params, d))
            assert abs(slope - dot) <= 1e-4 * (abs(slope) + 1)
        before = {i: (params[i].detach().double().clone(), opt.exp_avg[i].double().clone()) for i in mats}
        opt.all_reduce_grads()
        norm = opt.clip_grad_norm(1e6)
        assert math.isfinite(norm)
        opt.step()
        for i in mats:
            w, m = before[i]
            g = params[i].grad.double()
            m = 0.95 * m + 0.05 * g
            d = 1e-2 * 0.2 * math.sqrt(max(w.shape)) * definition(0.05 * g + 0.95 * m)
            err = float((params[i].detach().double() - (w - d)).norm())
            assert err <= NS * float(d.norm()) + 2.0 ** -23 * float(w.norm())


@pytest.mark.parametrize("budget", [1 << 32, 0], ids=["at_once", "one_by_one"])
def test_many_shapes_in_one_step(monkeypatch, budget):
    """More shapes than a run of the products takes, wide and tall, with sides up to 128 and beyond,
    that end in parts of blocks, in one pass through the workspace and in many."""
    import torch
    from hybridagent_b200 import ZeroOneMuon
    monkeypatch.setenv("HYBRIDAGENT_B200_MUON_BYTES", str(budget))
    shapes = [(255, 257), (130, 700), (700, 131), (64, 1000), (257, 255), (129, 200), (513, 300), (300, 513), (150, 2000),
              (255, 257), (20, 20), (641, 1300), (130, 700)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    params = [torch.nn.Parameter((torch.randn(s, generator=gen, device="cuda") * 0.02).bfloat16()) for s in shapes]
    opt = ZeroOneMuon([{"params": params, "lr": 2e-2}], rank=0, world_size=1, weight_decay=0.01)
    ref = Definition(opt, len(shapes), FACTORS["match_rms_adamw"])
    for step in range(2):
        set_grads(params, step, torch.bfloat16)
        norm = opt.clip_grad_norm(1.0)
        for i, p in enumerate(params):
            ref.step(i, p, 1.0 / (norm + 1e-6) if norm > 1.0 else None)
        opt.step()
    for i, p in enumerate(params):
        ref.check(i, opt, p, 2)


@pytest.mark.parametrize("seed", range(4))
def test_drawn_shapes(seed):
    """Sizes next to the tiles' and blocks' edges, twice each: the same bits, and the definition's values."""
    import random
    import torch
    from hybridagent_b200 import orthogonalize
    rng = random.Random(seed)
    edges = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 159, 160, 161, 191, 193, 255, 256, 257, 287, 289, 321, 383,
             385, 449, 511, 513, 639, 641, 767, 769, 1023, 1025]
    for _ in range(40):
        rows, cols = rng.choice(edges), rng.choice(edges)
        x = values("normal", (rng.choice([1, 2, 5]), rows, cols), torch.float32, seed=rows * 2000 + cols)
        y = orthogonalize(x)
        assert torch.equal(orthogonalize(x), y), (rows, cols)
        assert off(y, definition(x)) <= NS_BF16, (rows, cols)


def test_a_step_that_gave_up_is_reported():
    """What the weight kernel writes when a wait of the products ran out, here written by the host."""
    import torch
    params, opt, _ = build("small", torch.bfloat16)
    set_grads(params, 0, torch.bfloat16)
    opt.clip_grad_norm(1.0)
    opt.step()
    opt.state_dict()
    opt._muon_status[0] = 1
    with pytest.raises(RuntimeError, match="ran out"):
        opt.state_dict()
    set_grads(params, 1, torch.bfloat16)
    with pytest.raises(RuntimeError, match="ran out"):
        opt.step()


@pytest.mark.parametrize("shape", [(1, 383, 14575), (2, 11249, 366), (3, 2000, 140), (1, 742, 1520), (2, 260, 260),
                                   (35, 640, 1280), (20, 769, 1700), (24, 1600, 704), (30, 544, 352)])
def test_matrices_whose_singular_values_are_alike(shape):
    """They round the diagonals of all Gram matrices and factors the same way, unless those are kept.  What the fp16
    planes leave then, 2^-11 in elements of random sign, is less than the bf16 result's own rounding, 2^-8."""
    import torch
    from hybridagent_b200 import orthogonalize
    x = values("normal", shape, torch.float32, seed=sum(shape))
    want = definition(x)
    assert off(orthogonalize(x), want) <= 1.5 * off(want.bfloat16(), want)


def test_orthogonal_matrices_stay_so():
    import torch
    from hybridagent_b200 import orthogonalize
    for rows, cols in ((300, 300), (200, 1100), (1500, 700), (129, 5000)):
        x = torch.linalg.qr(values("normal", (max(rows, cols), min(rows, cols)), torch.float32, seed=rows))[0]
        x = (x if rows >= cols else x.mT).contiguous()
        assert off(orthogonalize(x), definition(x)) <= NS_BF16
