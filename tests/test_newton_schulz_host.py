"""Newton-Schulz products on the host: what the kernels' source, the library's own choices and the entry points' arguments have to hold, without a GPU."""
import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

from . import test_newton_schulz as ns

CSRC = Path(__file__).resolve().parent.parent / "mini_trainer_b200" / "csrc"


def body(source, name):
    """Text of a function, without its comments."""
    source = re.sub(r"//[^\n]*", "", source)
    at = source.index("{", source.index(") {", re.search(rf"\b{name}\(const", source).start()))
    depth = 0
    for i in range(at, len(source)):
        depth += {"{": 1, "}": -1}.get(source[i], 0)
        if depth == 0:
            return source[at:i]


@pytest.mark.parametrize("name", ["product_kernel", "split_kernel", "small_kernel"])
def test_warps_are_whole_before_aligned_instructions(name):
    """An instruction that is .aligned (allocation and loads of tensor memory, barriers of a cluster) is for warps whose threads come to it together, which nothing promises behind a block of one thread or
    a wait that each thread ends by itself: a barrier of the warp or the block has to be between."""
    together = r"__all_sync\(0xffffffffu, mbar_wait\(|__syncwarp\(\)|__syncthreads\(\)"
    apart = r"threadIdx\.x == 0\)|lane == 0\)|elect_one\(\)|mbar_wait\(|wait_sent\("
    aligned = r"cluster_barrier\(\)|tmem_alloc\(|tcgen05\.alloc|tmem_ld_\w+\(|tmem_dealloc\(|tcgen05\.dealloc"
    text, whole, seen = body((CSRC / "newton_schulz.cu").read_text(), name), True, 0
    for m in re.finditer(f"(?P<together>{together})|(?P<apart>{apart})|(?P<aligned>{aligned})", text):
        if m.lastgroup == "aligned":
            seen += 1
            assert whole, f"{name}: {text[max(0, m.start() - 300):m.end()]}"
        else:
            whole = m.lastgroup == "together"
    assert seen >= 5


def backend(name):
    from .test_native_host import make_ops
    if name == "plain":
        return TorchOps()
    ops = make_ops()
    ops.check_device = lambda t: None
    return ops


@pytest.mark.parametrize("name", ["plain", "native"])
@pytest.mark.parametrize("bad", [dict(scale=float("nan")), dict(scale=float("inf")), dict(grad_coef=float("nan")), dict(grad_coef=-float("inf"))])
def test_factors_that_are_not_finite_are_refused(name, bad):
    """They would overwrite the parameter, its momentum and its working copy with what is not finite."""
    ops, g = backend(name), torch.ones(6, 8)
    held = dict(master=g.clone(), moment=g.clone(), grad=g, param_out=g.bfloat16())
    with pytest.raises(ValueError, match="finite"):
        ops.muon_step(**held, lr=0.1, momentum=0.9, weight_decay=0.0, **bad)
    assert all((t == 1).all() for t in held.values())
    assert name == "plain" or not ops.calls


@pytest.mark.parametrize("name", ["plain", "native"])
def test_stacks_beyond_what_the_kernels_count_are_refused(name):
    ops = backend(name)
    for shape in ((1 << 24, 1, 1), (1 << 12, 1 << 12, 2, 3)):
        with pytest.raises(ValueError, match="more than the kernels count"):
            ops.orthogonalise(torch.empty(shape, device="meta"))


def calls(ops, shape, steps=5, muon=False):
    """Arguments of the library call that one of the entry points makes."""
    g = torch.ones(shape)
    if muon:
        ops.muon_step(g.clone(), g.clone(), g, g.bfloat16(), 0.1, 0.9, 0.0, steps=steps)
    else:
        ops.orthogonalise(g, steps)
    return ops.calls[-1]


@pytest.fixture
def current_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


@pytest.mark.parametrize("muon", [False, True])
def test_workspace_is_what_the_library_asks_for(current_device, muon):
    """None where the library makes the call one launch, which depends on the stack, the steps and the device too."""
    ops, asked = backend("native"), []

    def workspace(*sizes):
        asked.append(sizes)
        return 0 if sizes[2] == 3 else 4096 * sizes[3]
    ops._fn["mtb200_newton_schulz_workspace"] = workspace
    name, args = calls(ops, (3, 40, 24), 2, muon)
    assert name == ("mtb200_muon_step" if muon else "mtb200_newton_schulz") and asked == [(40, 24, 3, 2)] and args[-4:-2] == (None, 0)
    for steps in (2, 7):
        args = calls(ops, (4, 40, 24), steps, muon)[1]
        assert asked[-1] == (40, 24, 4, steps) and args[-4] and args[-3] == 4096 * steps


@pytest.fixture(scope="module")
def native():
    from mini_trainer_b200.ops import get_ops
    return get_ops(torch.device("cuda:0"))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 64), (64, 768, 16), (148, 128, 256), (32, 16384)])
def test_one_launch_holds_no_workspace(native, shape):
    assert native._fn["mtb200_newton_schulz_workspace"](*shape[-2:], math.prod(shape[:-2]), 5) == 0
    g = torch.randn(shape, device="cuda")
    native.orthogonalise(g)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = native.orthogonalise(g)
    assert torch.cuda.max_memory_allocated() - before <= out.numel() * 2 + 512   # the result alone, in the allocator's steps
    native.check_status()


@pytest.mark.parametrize("muon", [False, True])
def test_launches_are_counted_by_what_the_library_does(current_device, muon):
    """The backend's own count, of a stack of small matrices that is one launch and of one that is not."""
    ops, counted = backend("native"), []
    call = ops._call
    ops._call = lambda *a, n=1, tag=None: (counted.append(n), call(*a))
    ops._fn["mtb200_newton_schulz_workspace"] = lambda m, n, stack, steps: 0 if stack == 3 else 4096
    for shape, steps, more in (((3, 40, 24), 5, None), ((4, 40, 24), 5, 0), ((4, 40, 24), 2, 0), ((4, 24, 41), 5, 1), ((300, 300), 5, 1)):
        calls(ops, shape, steps, muon)
        assert counted.pop() == (1 if more is None else 2 + 3 * steps + (1 if muon else more))


def kernels_of(graph):
    """Number of a captured graph's nodes: all of these calls' are kernels."""
    n = ctypes.c_size_t()
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 64), (64, 128, 1024), (20, 128, 2048), (1000, 128, 256), (100, 601), (300, 301), (688, 256)])
@pytest.mark.parametrize("steps", [1, 5])
def test_launches_counted_are_launches_queued(native, shape, steps):
    g = torch.randn(shape, device="cuda") * 1e-3
    held = g.clone(), torch.zeros_like(g), g, g.bfloat16()
    for run in (lambda: native.orthogonalise(g, steps), lambda: native.muon_step(*held, 0.01, 0.9, 0.0, steps=steps)):
        run()
        graph, before = torch.cuda.CUDAGraph(keep_graph=True), native.launches
        with torch.cuda.graph(graph):
            kept = run()
        assert native.launches - before == kernels_of(graph)
        del kept
    native.check_status()


def scaled(shape, norm, kind="features", device="cpu", dtype=torch.float32):
    """Matrices of this norm each."""
    g = ns.matrices(kind, *shape, device=device).double()
    return (g / torch.linalg.matrix_norm(g, keepdim=True) * norm).to(dtype)


def large_matrices(ops, shape, device, tol):
    """Finite matrices whose squares are past the range of fp32: in a stack beside others, and a momentum of them."""
    for dtype in (torch.float32, torch.bfloat16):
        for norm in (1e18, 4e19, 1e25, 1e31, 1e38):
            g = scaled(shape, norm, device=device, dtype=dtype)
            ns.check(ops.orthogonalise(g), g, tol)
    g = torch.full(shape, 3e38, device=device)
    g[..., 0, ::2] *= -1.0
    ns.check(ops.orthogonalise(g), g, 3 * tol)   # (of rank two, with its rows alike: roundings in one direction)
    stack = torch.stack([scaled(shape, n, device=device) for n in (1.0, 1e30, 1e-3)])
    one = ops.orthogonalise(stack)
    ns.check(one, stack, tol)
    stack[1, ..., 0, 0] = float("inf")
    bad = ops.orthogonalise(stack)
    assert torch.equal(bad[0], one[0]) and torch.equal(bad[2], one[2]) and torch.isnan(bad[1]).any()
    g, w = scaled(shape, 1e25, device=device), torch.zeros(shape, device=device)
    ops.muon_step(w, torch.zeros_like(g), g, None, 1.0, 0.5, 0.0, nesterov=False, scale=1.0)
    want = -ns.exact(g)
    assert (torch.linalg.matrix_norm(w.double() - want) <= tol * torch.linalg.matrix_norm(want)).all()


@pytest.mark.parametrize("shape", [(13, 30), (40, 24), (2, 17, 9)])
def test_large_matrices_plain(shape):
    large_matrices(TorchOps(), shape, "cpu", 2.0 ** -10)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(13, 30), (40, 24), (128, 600), (2100, 100), (300, 520), (2, 264, 130), (301, 143)])
def test_large_matrices_by_the_kernels(native, shape):
    large_matrices(native, shape, "cuda", ns.TOL)
    native.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(13, 30), (128, 600), (2100, 100), (300, 520), (301, 143), (700, 1100)])
def test_norms_far_below_epsilon(native, shape):
    """An entry of X 2^p is held to half of fp16's smallest step, 2^-25, in the last two steps, which carry it on by 3.4445 each, and to 2^-36 in the others, by 485 at most: together 2^-25 (11.9 + 3.5 + 0.3) < 2^-21, so
    the result is off by 2^-21 sqrt(rows columns) / 2^p in norm at most, beside what it is off anyway; 2^p is within a factor of sqrt(2) of the root of the longer side."""
    for norm in (1e-8, 1e-11, 1e-13, 1e-15, 1e-18, 1e-30):
        g = scaled(shape, norm, device="cuda")
        got, want = native.orthogonalise(g).double(), ns.exact(g)
        off = (ns.TOL + ns.U / math.sqrt(3)) * want.norm() + 2.0 ** -21 * math.sqrt(2 * min(shape))
        assert float((got - want).norm()) <= float(off), norm
    native.check_status()
