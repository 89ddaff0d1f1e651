"""Cases of the Muon operators: what they are measured on, and their plain forms.

``orthogonalize``: five Newton-Schulz steps that push the singular values of a matrix (or of each
matrix of a batch) towards one.  With X0 = G / max(|G|_F, 1e-7) and m = min(rows, cols):

    A = X X^T,  X <- a X + (b A + c A A) X        (a, b, c) = (3.4445, -4.7750, 2.0315)

``step``: one training step of an optimizer over a parameter set whose matrices take the Muon
update and whose other tensors take AdamW's: global norm, clip, momentum with Nesterov's look-ahead,
orthogonalisation, decoupled decay, fp32 master and its rounded copy.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
A, B, C = 3.4445, -4.7750, 2.0315
STEPS, EPS = 5, 1e-7
MOMENTUM, DECAY, MAX_NORM = 0.95, 0.01, 1.0
B1, B2, ADAM_EPS = 0.9, 0.999, 1e-8
LR = 3e-5


# Parameter sets of the step cases: "m" matrices (rows, cols) that take the Muon update, "v" vectors.
SETS = {
    # a slice of the CPU configuration's set: launches and host work count
    "small": {"m": [(256, 512)] * 8 + [(1024, 256)] * 2, "v": [65536, 65536]},
    # one layer of the Qwen3-8B-shaped set
    "dense": {"m": [(4096, 4096), (1024, 4096), (1024, 4096), (4096, 4096), (12288, 4096), (12288, 4096),
                    (4096, 12288)], "v": [4096, 4096, 128, 128]},
    # part of a layer of the sparse set: attention, router, four experts
    "experts": {"m": [(4096, 2816), (2048, 2816), (2048, 2816), (2816, 4096), (128, 2816)] +
                     [(704, 2816), (704, 2816), (2816, 704)] * 4, "v": [2816]},
}


def listed():
    return [
        # one adapter-sized matrix: the latency of a call
        {"name": "one_64x96", "op": "orthogonalize", "batch": 1, "rows": 64, "cols": 96, "dtype": "bf16"},
        # the matrices of the CPU configuration, fp32 gradients
        {"name": "small_48x256x512", "op": "orthogonalize", "batch": 48, "rows": 256, "cols": 512, "dtype": "fp32"},
        {"name": "tall_8x1024x256", "op": "orthogonalize", "batch": 8, "rows": 1024, "cols": 256, "dtype": "fp32"},
        # sizes that fill no tile and whose rows start at any even address
        {"name": "odd_3x1000x1537", "op": "orthogonalize", "batch": 3, "rows": 1000, "cols": 1537, "dtype": "fp16"},
        # the gate projections of 128 experts
        {"name": "experts_128x704x2816", "op": "orthogonalize", "batch": 128, "rows": 704, "cols": 2816, "dtype": "bf16"},
        # one attention projection on its own: few tiles for the chip
        {"name": "square_4096x4096", "op": "orthogonalize", "batch": 1, "rows": 4096, "cols": 4096, "dtype": "bf16"},
        # one feed-forward projection of the 8B-shaped set
        {"name": "wide_4096x12288", "op": "orthogonalize", "batch": 1, "rows": 4096, "cols": 12288, "dtype": "bf16"},
        # the up and gate projections of the 14B-shaped set
        {"name": "tall_2x17408x5120", "op": "orthogonalize", "batch": 2, "rows": 17408, "cols": 5120, "dtype": "bf16"},
        # training steps: launch-bound, odd sizes in fp16, many small matrices, one dense layer
        {"name": "step_small_fp32", "op": "step", "set": "small", "dtype": "fp32"},
        {"name": "step_odd_fp16", "op": "step", "rows": 517, "cols": 1290, "count": 5, "vector": 4099, "dtype": "fp16"},
        {"name": "step_experts_bf16", "op": "step", "set": "experts", "dtype": "bf16"},
        {"name": "step_dense_bf16", "op": "step", "set": "dense", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
        rows, cols = _log(rng, 32, 17408), _log(rng, 32, 17408)
        if rng.random() < 0.5:  # half of them multiples of 64, as most weights are
            rows, cols = max(64, rows // 64 * 64), max(64, cols // 64 * 64)
        if rng.random() < 0.7:
            case = {"op": "orthogonalize", "batch": _log(rng, 1, 128), "rows": rows, "cols": cols, "dtype": dtype}
        else:
            case = {"op": "step", "rows": rows, "cols": cols, "count": _log(rng, 1, 12),
                    "vector": _log(rng, 1, 70000), "dtype": dtype}
        n = case["batch"] if case["op"] == "orthogonalize" else case["count"]
        if _flops(n, rows, cols) <= 1.2e13 and n * rows * cols <= 1.7e8:
            return case


def _tensors(case):
    """Shapes of a step case: matrices, then vectors."""
    if case.get("set"):
        s = SETS[case["set"]]
        return list(s["m"]), [(n,) for n in s["v"]]
    return [(case["rows"], case["cols"])] * case["count"], [(case["vector"],)]


def _gradient(gen, shape, dtype):
    """Gradients of about 1e-4 per element: a few strong directions over full-rank noise, for a matrix."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if len(shape) >= 2:
        left = torch.randn(*shape[:-1], 4, generator=gen, device="cuda")
        x += 0.5 * (left @ torch.randn(*shape[:-2], 4, shape[-1], generator=gen, device="cuda"))
    return (x * 1e-4).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "orthogonalize":
        return {"op": "orthogonalize", "x": _gradient(gen, (case["batch"], case["rows"], case["cols"]), dtype)}
    mats, vecs = _tensors(case)
    params, moms, vars_ = [], [], []
    for shape in mats + vecs:
        p = (torch.randn(shape, generator=gen, device="cuda") * 0.02).to(dtype)
        p = torch.nn.Parameter(p)
        p.grad = _gradient(gen, shape, dtype)
        params.append(p)
        moms.append(_gradient(gen, shape, torch.float32))
        vars_.append(torch.rand(shape, generator=gen, device="cuda") * 1e-8 if len(shape) == 1 else None)
    state = {"op": "step", "params": params, "n": len(mats)}
    if own:  # the optimizer that the program keeps, in the middle of a run
        from hybridagent_b200 import ZeroOneMuon
        opt = ZeroOneMuon([{"params": params[:len(mats)], "lr": LR},
                           {"params": params[len(mats):], "lr": LR, "use_muon": False}],
                          rank=0, world_size=1, weight_decay=DECAY)
        for i in range(len(params)):
            opt.exp_avg[i].copy_(moms[i])
            if vars_[i] is not None:
                opt.exp_avg_sq[i].copy_(vars_[i])
                opt.param_steps[i] = 100
        state["opt"] = opt
    else:  # fp32 parameters are their own masters
        state.update(master=[p.data if dtype == torch.float32 else p.data.float() for p in params], mom=moms,
                     var=vars_, steps=100)
    return state


def _orthogonal32(x):
    """The Newton-Schulz steps in 32 bits; x (..., rows, cols)."""
    x = x.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS).float()
    for _ in range(STEPS):
        g = x @ x.mT
        x = A * x + (B * g + C * (g @ g)) @ x
    return x.mT if tall else x


def _plain_step(s):
    params = s["params"]
    total = sum(p.grad.double().square().sum() for p in params)
    norm = total.sqrt()
    scale = torch.where(norm > MAX_NORM, MAX_NORM / (norm + 1e-6), 1.0).float()
    s["steps"] += 1
    for i, p in enumerate(params):
        g = (p.grad.float() * scale).to(p.dtype).float()  # clipped gradients are in the gradient's type
        w, m = s["master"][i], s["mom"][i]
        w.mul_(1 - LR * DECAY)
        if i < s["n"]:
            m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
            u = _orthogonal32((1 - MOMENTUM) * g + MOMENTUM * m)
            w.sub_(u, alpha=LR * 0.2 * math.sqrt(max(p.shape)))
        else:
            v = s["var"][i]
            m.mul_(B1).add_(g, alpha=1 - B1)
            v.mul_(B2).add_(g * g, alpha=1 - B2)
            w.sub_(LR * (m / (1 - B1 ** s["steps"])) / ((v / (1 - B2 ** s["steps"])).sqrt() + ADAM_EPS))
        if w is not p.data:
            p.data.copy_(w)
    return {"param": [p.data for p in params], "master": s["master"], "momentum": s["mom"], "variance": s["var"][s["n"]:]}


def run(state):
    if state["op"] == "orthogonalize":
        if own:
            from hybridagent_b200 import orthogonalize
            return orthogonalize(state["x"])
        return _orthogonal32(state["x"]).bfloat16()
    if not own:
        return _plain_step(state)
    opt = state["opt"]
    opt.all_reduce_grads()
    opt.clip_grad_norm(MAX_NORM)
    opt.step()
    k = range(len(state["params"]))
    return {"param": [p.data for p in state["params"]], "master": [opt.master[i] for i in k],
            "momentum": [opt.exp_avg[i] for i in k], "variance": [opt.exp_avg_sq[i] for i in k if i >= state["n"]]}


def _flops(n, rows, cols):
    """Products of the symmetric A and A A counted once for each pair of elements."""
    m, k = min(rows, cols), max(rows, cols)
    return n * STEPS * (3.0 * m * m * k + 1.0 * m ** 3)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "orthogonalize":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": n * (size + 2), "flops": _flops(case["batch"], case["rows"], case["cols"])}
    mats, vecs = _tensors(case)
    nm, nv = sum(r * c for r, c in mats), sum(n for n, in vecs)
    copy = 0 if size == 4 else size  # the low-precision copy of the parameter
    return {"bytes": nm * (size + 16 + copy) + nv * (size + 24 + copy),
            "flops": sum(_flops(1, r, c) for r, c in mats) + 10 * nm + 20 * nv}


def _exact_orthogonal(x):
    """In 64 bits, through the polynomial of the Gram matrix: U = S(G) X with S the product of the steps' factors."""
    x = x.double()
    if x.shape[-2] > x.shape[-1]:
        return _exact_orthogonal(x.mT).mT
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=EPS)
    gram = x @ x.mT
    one = torch.eye(gram.shape[-1], dtype=torch.float64, device=x.device)
    left = one
    for _ in range(STEPS):
        q = A * one + B * gram + C * (gram @ gram)
        left = q @ left
        gram = q @ gram @ q
    return left @ x


def exact(case, seed):
    if case["op"] == "orthogonalize":
        return _exact_orthogonal(prepare(case, seed)["x"])
    global own
    was, own = own, False  # the plain state holds the inputs, whichever side asks
    try:
        s = prepare(case, seed)
    finally:
        own = was
    norm = math.sqrt(sum(float(p.grad.double().pow(2).sum()) for p in s["params"]))
    scale = MAX_NORM / (norm + 1e-6) if norm > MAX_NORM else 1.0
    t = s["steps"] + 1
    out = {"param": [], "master": [], "momentum": [], "variance": []}
    for i, p in enumerate(s["params"]):
        g = (p.grad.double() * scale).to(p.dtype).double()
        w, m = s["master"][i].double() * (1 - LR * DECAY), s["mom"][i].double()
        if i < s["n"]:
            m = MOMENTUM * m + (1 - MOMENTUM) * g
            w = w - LR * 0.2 * math.sqrt(max(p.shape)) * _exact_orthogonal(MOMENTUM * m + (1 - MOMENTUM) * g)
        else:
            m = B1 * m + (1 - B1) * g
            v = B2 * s["var"][i].double() + (1 - B2) * g * g
            w = w - LR * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + ADAM_EPS)
            out["variance"].append(v)
        out["param"].append(w)
        out["master"].append(w)
        out["momentum"].append(m)
    return out
