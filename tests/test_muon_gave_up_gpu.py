"""What a call leaves behind when a wait inside its products ran out.

No wait runs out here: the calls are captured into graphs, and a node between two kernels sets the workspace's error
word, as a CTA that gave up does.  All kernels run to their ends and act on the word as they would on a real one."""
import ctypes

import numpy as np
import pytest

from hybridagent_b200 import _lib, muon

pytestmark = pytest.mark.gpu


def check(result):
    from cuda.bindings import runtime as rt
    assert result[0] == rt.cudaError_t.cudaSuccess, result[0]
    return result[1:]


def with_error_word(call, workspace, before):
    """Captures call() and replays it with a node that sets the first word of the workspace before kernel `before` (counted
    from the end) of its chain."""
    import torch
    from cuda.bindings import runtime as rt
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = rt.cudaGraph_t(int(graph.raw_cuda_graph()))
    count = check(rt.cudaGraphGetNodes(raw))[-1]
    nodes = check(rt.cudaGraphGetNodes(raw, count))[0][:count]
    edges = check(rt.cudaGraphGetEdges_v2(raw))[-1]
    sources, targets, data = (list(x)[:edges] for x in check(rt.cudaGraphGetEdges_v2(raw, edges))[:3])
    chain = [n for n in nodes if int(n) not in {int(t) for t in targets}]
    assert len(chain) == 1 and edges == count - 1
    after = {int(s): (t, d) for s, t, d in zip(sources, targets, data)}
    while int(chain[-1]) in after:
        chain.append(after[int(chain[-1])][0])
    first, second = chain[-before - 1], chain[-before]
    check(rt.cudaGraphRemoveDependencies_v2(raw, [first], [second], [after[int(first)][1]], 1))
    params = rt.cudaMemsetParams()
    params.dst, params.value, params.elementSize, params.width, params.height = workspace.data_ptr(), 1, 4, 1, 1
    node, = check(rt.cudaGraphAddMemsetNode(raw, [first], 1, params))
    check(rt.cudaGraphAddDependencies(raw, [node], [second], 1))
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    return len(chain)


@pytest.mark.parametrize("shape", [(1, 64, 96), (3, 64, 96), (2, 128, 2816), (5, 9000, 32), (3, 300, 400), (2, 512, 256),
                                   (1, 1500, 2304), (2, 300, 397), (3, 40, 61)], ids=lambda s: "x".join(map(str, s)))
def test_the_whole_result_is_nan(shape):
    """Where the products store the result themselves and where a kernel behind them does."""
    import torch
    n, rows, cols = shape
    x = torch.randn(shape, device="cuda").bfloat16()
    out = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    ns = muon._ns_params(5, muon.COEFFICIENTS, 1e-7)
    size = muon._workspace_bytes(n, rows, cols)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def call():
        _lib.call("ha_orthogonalize", x.data_ptr(), _lib.HA_BF16, out.data_ptr(), n, rows, cols, ctypes.byref(ns),
                  ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)

    call()
    torch.cuda.synchronize()
    assert out.isfinite().all()
    out.zero_()
    with_error_word(call, ws, 1)
    assert out.isnan().all()
    call()  # the next call starts afresh
    torch.cuda.synchronize()
    assert out.isfinite().all()


@pytest.mark.parametrize("rows,cols", [(64, 96), (300, 400)])
def test_a_step_leaves_the_weights_and_sets_the_status(rows, cols):
    import torch
    grad = torch.randn(rows, cols, device="cuda").bfloat16()
    master, moment = torch.randn(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
    param = master.bfloat16()
    tab = np.zeros(1, dtype=_lib.TENSOR_DTYPE)
    for name, value in (("grad", grad.data_ptr()), ("master", master.data_ptr()), ("exp_avg", moment.data_ptr()),
                        ("param", param.data_ptr()), ("numel", rows * cols), ("decay", 0.5), ("neg_lr", -1e-2)):
        tab[name] = value
    shapes = np.asarray([[rows, cols]], dtype=np.int64)
    sc = _lib.MuonScalars(0.95, 0.05, 1, 1, 0, 1.0)
    ns = muon._ns_params(5, muon.COEFFICIENTS, 1e-7)
    size = muon._workspace_bytes(1, rows, cols)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call():
        _lib.call("ha_muon_step", _lib.np_ptr(tab), _lib.np_ptr(shapes), 1, _lib.HA_BF16, ctypes.byref(sc), ctypes.byref(ns), 0,
                  None, None, status.data_ptr(), ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)

    before = master.clone(), param.clone()
    for kernel in (1, 2):  # the word is set before the weights' kernel, and before the products
        moment.zero_()
        status.zero_()
        with_error_word(call, ws, kernel)
        assert int(status) == 1
        assert torch.equal(master, before[0]) and torch.equal(param, before[1])
        assert moment.abs().max() > 0  # the momentum has been updated


def test_the_optimizer_raises_before_anything_changes_until_a_state_is_loaded():
    import torch
    from hybridagent_b200 import ZeroOneMuon
    gen = torch.Generator(device="cuda").manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda").bfloat16()) for s in [(40, 60), (300, 280), (99,)]]
    opt = ZeroOneMuon([{"params": params, "lr": 1e-2}], rank=0, world_size=1)

    def grads():
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen, device="cuda").bfloat16()

    grads()
    opt.clip_grad_norm(1.0)
    opt.step()
    good = opt.state_dict()
    grads()
    opt.clip_grad_norm(0.5)
    opt._muon_status[0] = 1  # as the weights' kernel writes it
    counts, clip = dict(opt.param_steps), opt._pending_clip
    weights, moments = [p.detach().clone() for p in params], [opt.exp_avg[i].clone() for i in range(3)]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="ran out"):
            opt.step()
        assert opt.step_count == 1 and dict(opt.param_steps) == counts and opt._pending_clip == clip is not None
    with pytest.raises(RuntimeError, match="ran out"):
        opt.state_dict()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(weights, params))
    assert all(torch.equal(m, opt.exp_avg[i]) for i, m in enumerate(moments))
    opt.load_state_dict(good)
    grads()
    opt.clip_grad_norm(1.0)
    opt.step()
    assert opt.state_dict()["step_count"] == 2
