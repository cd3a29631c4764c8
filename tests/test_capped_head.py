"""LM head and cross-entropy on logits capped by a tanh, on the CPU and by the kernels, against 64 bits.

Tolerances count roundings. The products z = x w come in fp32: off by at most 2^-17 of sum |x w| (sums of up to 4096 terms, added up in blocks). A capped logit is off by 5.1e-7 of
itself within the cap and 2^-21 of the cap beyond it (and for caps over 2048), and by the product's error; the loss by those of its target and of the others on average, and
by 2^-18 of the logits' size. The gradient is formed from l / cap rounded to fp16 (2^-11), and rounded to bf16 once (U = 2^-8) before the products that dx and dw are, which are rounded once more."""
import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

U = torch.finfo(torch.bfloat16).eps / 2
H = torch.finfo(torch.float16).eps / 2
IGNORE = -100


def inputs(T, H, V, gain=3.0, seed=0, device="cpu", ignored=0.25):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(T, H, generator=g).bfloat16(), (torch.randn(V, H, generator=g) * gain / H ** 0.5).bfloat16()
    t = torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) < ignored] = IGNORE
    return x.to(device), w.to(device), t.to(device)


def exact(x, w, t, cap, scale, grad_scale):
    """``(values, bounds)`` of loss, dx and dw."""
    x, w, t = x.double().cpu(), w.double().cpu(), t.cpu()
    z = x @ w.t() * scale
    th = torch.tanh(z / cap)
    l, c = cap * th, 1 - th * th
    ez = 2.0 ** -17 * (x.abs() @ w.abs().t()) * abs(scale)
    el = c * ez + 5.1e-7 * l.abs() + 2.0 ** -21 * cap * ((z.abs() > cap) | (cap > 2048)) + 2.0 ** -22 * l.abs()
    p, valid, safe = torch.softmax(l, 1), t != IGNORE, t.clamp_min(0)[:, None]
    one = torch.zeros_like(p).scatter_(1, safe, 1.0)
    loss = torch.where(valid, torch.logsumexp(l, 1) - l.gather(1, safe)[:, 0], 0.0)
    mean = (p * el).sum(1)
    bl = valid * (mean + el.gather(1, safe)[:, 0] + 2.0 ** -18 * l.abs().amax(1) + 2.0 ** -20)
    dz = (p - one) * c * (valid * grad_scale)[:, None]
    # t = l / cap is rounded to fp16, H of itself or 2^-25 below its normal numbers: the exponential is off by the logit's error, the derivative 1 - t^2 by 2 |t| dt
    et = H * th.abs().clamp_min(2.0 ** -14)
    edz = U * dz.abs() + (1.02 * p * (el + mean[:, None] + cap * et + 2.0 ** -18) * c + (p - one).abs() * (2 * th.abs() * et + et * et + 2 * el.clamp_max(cap) / cap + 2.0 ** -21)) \
        * (valid * abs(grad_scale))[:, None]
    dx, dw = dz @ w * scale, dz.t() @ x * scale
    bx, bw = (1.01 * edz + 2.0 ** -17 * dz.abs()) @ w.abs() * abs(scale), (1.01 * edz + 2.0 ** -17 * dz.abs()).t() @ x.abs() * abs(scale)
    return (loss, dx, dw), (bl, bx + U * dx.abs() + 1e-30, bw + U * dw.abs() + 1e-30)


def run(ops, x, w, t, cap, scale, grad_scale, dw=None, accumulate=False):
    dw = torch.full_like(w, float("nan")) if dw is None else dw
    loss, dx = ops.linear_ce(x, w, t, grad_scale, dw, accumulate_dw=accumulate, logit_scale=scale, softcap=cap)
    return loss, dx, dw


def check(ops, *args):
    got, (want, bound) = run(ops, *args), exact(*args)
    for name, g, v, b in zip(("loss", "dx", "dw"), got, want, bound):
        over = (g.double().cpu() - v).abs() - b
        assert torch.isfinite(g).all() and over.max() <= 0, (name, int((over > 0).sum()), float(over.max()))
    return got


# ------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("cap,gain,scale", [(30.0, 3.0, 1.0), (2.0, 3.0, 1.0), (15.0, 100.0, 0.5), (0.01, 1.0, 2.0)])
def test_plain_backend_against_64_bits(cap, gain, scale):
    for T, H, V in ((1, 8, 8), (7, 24, 40), (33, 64, 264)):
        check(TorchOps(ce_chunk=16), *inputs(T, H, V, gain, seed=V), cap, scale, 1.0 / T)


def test_formula_against_differences():
    """The summed loss along a direction of x and w, by central differences in 64 bits with a step of 2^-20."""
    x, w, t = inputs(9, 32, 72)
    u, v = (torch.randn(a.shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64) for k, a in ((1, x), (2, w)))
    (_, dx, dw), _ = exact(x, w, t, 4.0, 1.0, 1.0)
    f = [exact(x.double() + e * u, w.double() + e * v, t, 4.0, 1.0, 1.0)[0][0].sum() for e in (2.0 ** -20, -2.0 ** -20)]
    want = (dx * u).sum() + (dw * v).sum()
    assert abs((f[0] - f[1]) / 2.0 ** -19 - want) <= 1e-8 * ((dx * u).abs().sum() + (dw * v).abs().sum())


def test_a_high_cap_is_no_cap():
    x, w, t = inputs(20, 32, 72)
    dw = torch.empty_like(w)
    loss, dx = TorchOps().linear_ce(x, w, t, 0.1, dw)
    a, b, c = run(TorchOps(), x, w, t, 1e4, 1.0, 0.1)
    assert torch.allclose(a, loss, atol=1e-4) and torch.allclose(b.float(), dx.float(), atol=1e-2 * dx.float().abs().max()) and torch.allclose(c.float(), dw.float(), atol=1e-2 * dw.float().abs().max())
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="cap"):
            run(TorchOps(), x, w, t, bad, 1.0, 0.1)


def test_calls_of_the_kernels_and_their_refusals():
    from .test_native_host import make_ops
    ops = make_ops()
    ops.ce_chunk, ops._index = 64, None
    x, w, t = inputs(70, 32, 72)
    dw = torch.empty_like(w)
    ops.linear_ce(x, w, t, 0.1, dw, logit_scale=0.5, softcap=30.0)   # two chunks: products, loss, two gradients each, the sum of dw rounded at the end
    names = [n for n, _ in ops.calls]
    assert names[:2] == names[4:6] == ["mtb200_gemm_capped", "mtb200_ce_capped"] and names[-1] == "mtb200_f32_to_bf16" and len(names) == 9
    assert [a[6:11] for n, a in ops.calls if n == "mtb200_ce_capped"] == [(k, 72, 32, 0.5 / 30.0, 30.0 * 1.4426950408889634) for k in (64, 6)]
    n = len(ops.calls)
    dw.fill_(1.0)
    loss, dx = ops.linear_ce(x[:0], w, t[:0], 0.1, dw, accumulate_dw=True, softcap=30.0)
    assert loss.shape == (0,) and dx.shape == (0, 32) and dw.min() == 1.0
    ops.linear_ce(x[:0], w, t[:0], 0.1, dw, softcap=30.0)
    assert not dw.any()
    for args in ((x.float(), w, t, dw), (x[:, :24], w, t, dw), (x, w[:, :24].contiguous(), t, dw), (x, w[:36], t, dw[:36]), (x, w, t[:50], dw), (x, w, t.int(), dw),
                 (x, w, t, dw[:36]), (x, w, t, dw.float()), (x.t().contiguous().t(), w, t, dw), (x, w, torch.stack([t, t], 1)[:, 0], dw)):
        with pytest.raises(ValueError):
            ops.linear_ce(args[0], args[1], args[2], 0.1, args[3], softcap=30.0)
    for cap in (0.0, -2.0, 1e9, 1e-9, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="capped at"):
            ops.linear_ce(x, w, t, 0.1, dw, softcap=cap)
    assert len(ops.calls) == n


def test_choice_of_the_product():
    from mini_trainer_b200.ops import gemm_plan
    assert [gemm_plan.capped_form(*c, False, 74) for c in ((3720, 1536), (128, 4096), (5000, 512))] == [1, 0, 0]
    assert gemm_plan.capped_form(3720, 1536, True, 0) == 0 and gemm_plan.capped_form(100, 64, True, 74) == 1


# ------------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("cap,gain,scale", [(30.0, 3.0, 1.0), (2.0, 3.0, 1.0), (15.0, 100.0, 0.5), (4096.0, 3.0, 1.0), (0.01, 1.0, 1.0)])
@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("T,H,V", [(1, 8, 8), (5, 64, 264), (129, 72, 1000), (33, 256, 8200), (300, 512, 4096), (17, 128, 40008), (257, 1032, 520)])
def test_kernels_against_64_bits(ops, T, H, V, cap, gain, scale, pair, monkeypatch):
    from mini_trainer_b200.ops import gemm_plan
    monkeypatch.setattr(gemm_plan, "capped_form", lambda *a: pair)
    check(ops, *inputs(T, H, V, gain, seed=T, device="cuda"), cap, scale, 1.0 / T)
    ops.check_status()


@pytest.mark.gpu
def test_chunks_accumulation_and_ignored_rows():
    from mini_trainer_b200.ops.native import NativeOps
    ops = NativeOps("cuda:0", ce_chunk=128)
    x, w, t = inputs(300, 128, 1032, device="cuda")
    loss, dx, dw = check(ops, x, w, t, 25.0, 0.8, 0.01)
    assert not loss[t == IGNORE].any() and not dx[t == IGNORE].any()
    again = run(ops, x, w, t, 25.0, 0.8, 0.01, dw=dw.clone(), accumulate=True)[2]
    assert ((again.float() - 2 * dw.float()).abs() <= 2.1 * U * again.float().abs() + 1e-30).all()
    t[:] = IGNORE
    loss, dx, dw = run(ops, x, w, t, 25.0, 0.8, 0.01)
    assert not loss.any() and not dx.any() and not dw.any()
    t[:] = 1032   # no column: reported in the loss, as without a cap
    assert torch.isnan(run(ops, x, w, t, 25.0, 0.8, 0.01)[0]).all()
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(1, 4096), (2, 8192), (3, 8200), (7, 20008), (7, 65544), (300, 16392)])
def test_rows_divided_over_blocks(ops, T, V):
    """Targets in every part of a row, at the first and last column; ignored rows are zero in all of their parts, and a target that is no column is one row's."""
    x, w, t = inputs(T, 64, V, seed=V, device="cuda")
    t.copy_(torch.linspace(V - 1, 0, T).round().long() if T > 1 else torch.tensor([V - 1]))
    check(ops, x, w, t, 30.0, 1.0, 1.0 / T)
    t[T // 2] = IGNORE
    loss, dx, dw = check(ops, x, w, t, 30.0, 1.0, 1.0 / T)
    assert loss[T // 2] == 0 and not dx[T // 2].any()
    t[T // 2] = V
    again = run(ops, x, w, t, 30.0, 1.0, 1.0 / T)[0]
    assert torch.isnan(again[T // 2]) and torch.equal(torch.isnan(again).nonzero().flatten(), torch.tensor([T // 2], device="cuda"))
    ops.check_status()


@pytest.mark.gpu
def test_captured_on_two_streams_and_twice(ops):
    x, w, t = inputs(200, 256, 2048, device="cuda")
    a = run(ops, x, w, t, 30.0, 1.0, 0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(ops, x, w, t, 30.0, 1.0, 0.01)
    c = run(ops, x, w, t, 30.0, 1.0, 0.01)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a, b, c))
    graph, dw = torch.cuda.CUDAGraph(), torch.empty_like(w)
    with torch.cuda.graph(graph):
        out = run(ops, x, w, t, 30.0, 1.0, 0.01, dw=dw)
    nx, nw, nt = inputs(200, 256, 2048, seed=9, device="cuda")
    x.copy_(nx), w.copy_(nw), t.copy_(nt)
    graph.replay()
    torch.cuda.synchronize()
    want, bound = exact(nx, nw, nt, 30.0, 1.0, 0.01)
    for g, v, e in zip(out, want, bound):
        assert ((g.double().cpu() - v).abs() <= e).all()
    ops.check_status()
