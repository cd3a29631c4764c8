"""Arguments of ``linear_nll`` and its gradient at the edges of what is documented: memory that is shared, targets outside the vocabulary, what a captured call takes."""
import ctypes

import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps


def arguments(T=6, H=16, V=24):
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(T, H, generator=g).bfloat16(), torch.randn(V, H, generator=g).bfloat16()
    one = torch.ones(T)
    return dict(dloss=one.clone(), x=x, w=w, targets=torch.randint(0, V, (T,), generator=g), loss=one.clone(), lse=one.clone(), dlse=one.clone(), dw_out=torch.empty_like(w))


@pytest.mark.parametrize("backend", ["plain", "native"])
@pytest.mark.parametrize("name,shift", [("w", 0), ("w", 1), ("w", 23), ("w", -1), ("w", -23), ("x", 1), ("x", -5), ("x", 23), ("dloss", 0), ("loss", 0), ("lse", 0), ("dlse", 0), ("targets", 0)])
def test_weight_gradient_over_an_operand_is_refused(backend, name, shift):
    """A part of the weight that is overwritten would be read by the pieces of the vocabulary behind it."""
    from .test_native_host import make_ops
    ops = TorchOps() if backend == "plain" else make_ops()
    if backend == "native":
        ops.check_device = lambda t: None
    v = arguments()
    rows = v["w"].shape[0]
    memory = torch.zeros(3 * rows, v["w"].shape[1], dtype=torch.bfloat16)
    dw = memory[rows:2 * rows]
    if name in ("w", "x"):
        v[name] = memory[rows + shift:][:v[name].shape[0]].copy_(v[name])
    else:
        n = v[name].numel() * v[name].element_size()
        v[name] = dw.view(-1).view(torch.uint8)[64:64 + n].view(v[name].dtype).copy_(v[name])
    with pytest.raises(ValueError, match="memory of its own"):
        ops.linear_nll_bwd(**{**v, "dw_out": dw})
    if backend == "native":
        assert not ops.calls


@pytest.mark.parametrize("shift", [24, -24])
def test_weight_gradient_beside_an_operand(shift):
    """Neighbours in one allocation, as parameters and their gradients are, share nothing."""
    v = arguments()
    memory = torch.zeros(72, 16, dtype=torch.bfloat16)
    v["w"], dw = memory[24 + shift:48 + shift].copy_(v["w"]), memory[24:48]
    dx = TorchOps().linear_nll_bwd(**{**v, "dw_out": dw})
    want = torch.empty_like(v["w"])
    assert torch.equal(dx, TorchOps().linear_nll_bwd(**{**v, "dw_out": want})) and torch.equal(dw, want)


def targets_outside(ops, device, dtype):
    """A target that is no column counts as ignored, in the losses and in both gradients, and is reported once."""
    g = torch.Generator().manual_seed(1)
    T, H, V = 40, 16, 5
    x, w = torch.randn(T, H, generator=g).to(dtype).to(device), torch.randn(V, H, generator=g).to(dtype).to(device)
    t = torch.randint(0, V, (T,), generator=g).to(device)
    t[3] = -100
    dloss, dlse = torch.randn(T, generator=g).to(device), torch.randn(T, generator=g).to(device)
    ignored, outside = t.clone(), t.clone()
    rows = torch.tensor([0, 7, 8, 30, 39], device=device)
    ignored[rows] = -100
    outside[rows] = torch.tensor([V, -1, 1 << 40, -(1 << 62), V + 3], device=device)

    def run(targets):
        loss, lse = ops.linear_nll(x, w, targets)
        dw = torch.empty_like(w)
        return loss, lse, ops.linear_nll_bwd(dloss, x, w, targets, loss, lse, dw, dlse=dlse), dw
    want = run(ignored)
    ops.check_status()
    assert (want[0][rows] == 0).all() and (want[2][rows] == 0).all() and (want[0][[1, 2, 4]] > 0).all()
    got = run(outside)
    run(t)   # a call without such targets takes nothing back
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="target outside the vocabulary"):
        ops.check_status()
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_targets_outside_the_vocabulary(dtype):
    targets_outside(TorchOps(ce_chunk=11), "cpu", dtype)


@pytest.mark.gpu
def test_targets_outside_the_vocabulary_by_the_kernels():
    from mini_trainer_b200.ops import get_ops
    targets_outside(get_ops(torch.device("cuda:0")), "cuda", torch.bfloat16)


@pytest.mark.parametrize("capturing", [False, True])
def test_arrival_counters_are_made_where_a_product_splits(monkeypatch, capturing):
    """Under capture a call has counters of its own, one set for all of its products that split and none where none does; outside of a graph a stream's are used."""
    from .test_native_host import make_ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    made, zeros = [], torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: made.append(a) or zeros(*a, **k))
    ops = make_ops()
    ops.check_device = lambda t: None
    stream = zeros(1, dtype=torch.int64)
    ops._split_workspace = lambda st: stream
    for T, H, V, splits in ((6, 16, 24, False), (64, 256, 30016, True), (64, 1024, 30016, True)):
        v = arguments(T, H, V)
        made.clear(), ops.calls.clear()
        ops.linear_nll_bwd(**v)
        products = [a for n, a in ops.calls if n.startswith("mtb200_gemm") and n != "mtb200_gemm_nll"]
        divided = [a for a in products if a[16] > 1]
        assert len(products) == 2 and bool(divided) == splits
        assert len(made) == (capturing and splits)
        own = {a[17] for a in divided}
        assert len(own) == splits and all((a == stream.data_ptr()) != capturing for a in own)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,splits", [(5, 64, 500, False), (64, 1024, 30016, True)])
def test_a_captured_gradient_is_its_launches(T, H, V, splits):
    """Nothing in the graph beside the kernels, and one set of counters where a product splits."""
    from mini_trainer_b200.ops import get_ops
    ops = get_ops(torch.device("cuda:0"))
    v = {k: t.cuda() for k, t in arguments(T, H, V).items()}
    ops.linear_nll_bwd(**v)
    graph, before, n = torch.cuda.CUDAGraph(keep_graph=True), ops.launches, ctypes.c_size_t()
    with torch.cuda.graph(graph):
        held = ops.linear_nll_bwd(**v)
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    assert n.value == ops.launches - before + splits and held.shape == v["x"].shape
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V", [(300, 256, 5000), (64, 1024, 30016), (700, 512, 9001), (1, 64, 40000)])
def test_replays_are_the_calls_outside_of_a_graph(T, H, V):
    """Losses and gradients bit for bit, products that split their reduction among them."""
    from mini_trainer_b200.ops import get_ops
    ops = get_ops(torch.device("cuda:0"))
    v = {k: t.cuda() for k, t in arguments(T, H, V).items()}
    v["targets"][::5] = -100

    def run():
        loss, lse = ops.linear_nll(v["x"], v["w"], v["targets"])
        dw = torch.empty_like(v["w"])
        return loss, lse, ops.linear_nll_bwd(v["dloss"], v["x"], v["w"], v["targets"], loss, lse, dw, dlse=v["dlse"]), dw
    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(2):
        for t in held:
            t.fill_(7)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    ops.check_status()
