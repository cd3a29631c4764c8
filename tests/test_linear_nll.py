"""Likelihoods without logits (``linear_nll`` and its gradient), on the CPU and by the kernels, against 64 bits.

Tolerances count roundings. A logit is an fp32 sum of H products of bf16 numbers, added in blocks of at least 8: off by at most (H / 8 + 8) 2^-23 of the sum of
their absolute values, D below. The log-partition is off by that, two units of the exponential and a chain of sums (2^-18 together, of terms below one), and a rounding of itself; the loss by two logits' worth. A
logit's gradient is off by twice D + 2^-17 of itself (the logit and the log-partition in its exponent) and a rounding to bf16, U = 2^-8, as an operand; the sums over it once more by U in their
storage and by their fp32 chain."""
import pytest
import torch

from mini_trainer_b200.ops import linear_nll as LN
from mini_trainer_b200.ops.torch_ref import TorchOps

U = torch.finfo(torch.bfloat16).eps / 2
IGN = -100


def inputs(T, H, V, ignored=0.2, gain=3.0, seed=0, device="cpu", dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(T, H, generator=g).to(dtype), (torch.randn(V, H, generator=g) * gain / H ** 0.5).to(dtype)
    t = torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) < ignored] = IGN
    v = {"x": x, "w": w, "t": t, "dloss": torch.randn(T, generator=g), "dlse": torch.randn(T, generator=g)}
    return {k: a.to(device) for k, a in v.items()}


def check(ops, v, scale=1.0, z=True, accumulate=False, out_unit=U, operand_unit=U):
    x, w, t = v["x"], v["w"], v["t"]
    (T, H), V = x.shape, w.shape[0]
    loss, lse = ops.linear_nll(x, w, t, logit_scale=scale)
    assert loss.dtype == lse.dtype == torch.float32 and loss.shape == lse.shape == (T,)
    xd, wd = x.double(), w.double()
    logits = xd @ wd.t() * scale
    D = (H / 8 + 8) * 2.0 ** -23 * abs(scale) * (xd.abs() @ wd.abs().t()).amax(1) if T else torch.zeros(0, device=x.device)
    ok = t != IGN
    want_lse = torch.logsumexp(logits, 1)
    want = torch.where(ok, want_lse - logits.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0)
    small = 2.0 ** -18 + 2.0 ** -22 * (want_lse.abs() + logits.abs().amax(1))
    assert ((lse - want_lse).abs() <= D + small).all()
    assert ((loss - want).abs() <= 2 * D + 2 * small).all() and (loss[~ok] == 0).all()
    # gradients
    before = torch.randn(V, H, device=x.device).to(w.dtype)
    dw = before.clone()
    dx = ops.linear_nll_bwd(v["dloss"], x, w, t, loss, lse, dw, accumulate_dw=accumulate, logit_scale=scale, dlse=v["dlse"] if z else None)
    dl = torch.where(ok, v["dloss"].double(), 0.0)
    dz = torch.where(ok, v["dlse"].double(), 0.0) if z else torch.zeros_like(dl)
    p = torch.softmax(logits, 1)
    hot = torch.zeros_like(p).scatter_(1, t.clamp_min(0)[:, None], 1.0)
    g = p * (dl + dz)[:, None] - hot * dl[:, None]
    mag = p * (dl + dz).abs()[:, None] + hot * ((1 - p) * dl.abs()[:, None] + p * dz.abs()[:, None])
    off = abs(scale) * mag * (operand_unit + 2 * D + 2 * small + 2.0 ** -17)[:, None]
    want_dx, want_dw = scale * g @ wd, scale * g.t() @ xd
    if accumulate:
        want_dw = want_dw + before.double()
    chain = lambda n: (n / 8 + 16) * 2.0 ** -23
    assert ((dx.double() - want_dx).abs() <= out_unit * want_dx.abs() + (1 + out_unit) * (off + chain(V) * abs(scale) * mag) @ wd.abs() + 1e-30).all()
    assert ((dw.double() - want_dw).abs() <= out_unit * want_dw.abs() + (1 + out_unit) * ((off + chain(T) * abs(scale) * mag).t() @ xd.abs() + 2.0 ** -23 * want_dw.abs()) + 1e-30).all()
    assert (dx[~ok] == 0).all()
    return loss, lse, dx, dw


CASES = [(1, 8, 1), (1, 64, 2), (7, 264, 127), (129, 64, 129), (33, 128, 1000), (130, 520, 515)]


@pytest.mark.parametrize("T,H,V", CASES)
@pytest.mark.parametrize("z,accumulate,scale", [(True, False, 1.0), (False, True, 0.3)])
def test_plain_form(T, H, V, z, accumulate, scale):
    check(TorchOps(), inputs(T, H, V), scale, z, accumulate)
    check(TorchOps(ce_chunk=11), inputs(T, H, V, dtype=torch.float32), scale, z, accumulate, out_unit=2.0 ** -23, operand_unit=2.0 ** -20)


def test_gradient_against_differences():
    v = inputs(5, 8, 13, dtype=torch.float32)
    ops, x, w, t = TorchOps(), v["x"], v["w"], v["t"]
    loss, lse = ops.linear_nll(x, w, t)
    dw = torch.empty_like(w)
    dx = ops.linear_nll_bwd(v["dloss"], x, w, t, loss, lse, dw, dlse=v["dlse"])
    ok = t != IGN

    def f(a, b):
        z = a @ b.t()
        l = torch.logsumexp(z, 1)
        return float(((l - z.gather(1, t.clamp_min(0)[:, None])[:, 0]) * v["dloss"].double() + l * v["dlse"].double())[ok].sum())
    for grad, name in ((dx, "x"), (dw, "w")):
        for i in range(0, grad.numel(), 7):
            h = torch.zeros(grad.numel(), dtype=torch.float64)
            h[i] = 1e-5
            h = h.view(grad.shape)
            a, b = x.double(), w.double()
            d = (f(a + h, b) - f(a - h, b)) if name == "x" else (f(a, b + h) - f(a, b - h))
            assert abs(d / 2e-5 - float(grad.reshape(-1)[i])) < 1e-5


def test_sum_of_losses_is_linear_ce():
    """One uniform weight is what ``linear_ce`` computes."""
    v, ops = inputs(40, 32, 77, dtype=torch.float32), TorchOps()
    loss, lse = ops.linear_nll(v["x"], v["w"], v["t"])
    dw, dw2 = torch.empty_like(v["w"]), torch.empty_like(v["w"])
    dx = ops.linear_nll_bwd(torch.full((40,), 0.25), v["x"], v["w"], v["t"], loss, lse, dw)
    want, dx2 = ops.linear_ce(v["x"], v["w"], v["t"], 0.25, dw2)
    assert torch.allclose(loss, want, atol=1e-5) and torch.allclose(dx, dx2, atol=1e-5) and torch.allclose(dw, dw2, atol=1e-5)


def test_pieces():
    """Pieces cover the vocabulary in whole tiles, in as few as their bytes allow, within them where two tiles allow it."""
    for T in (1, 2, 127, 1777, 8192, 64000, 1 << 20):
        for V in (1, 255, 257, 512, 32000, 50021, 128256, 151936):
            n = LN.piece_columns(T, V)
            assert 1 <= n <= V and (n == V or n % 256 == 0)
            assert n * T * 2 <= LN.PIECE_BYTES or n <= 512 or n == V == 1
            assert -(-V // n) <= -(-V // max(512, LN.PIECE_BYTES // 2 // T // 256 * 256))


@pytest.mark.parametrize("backend", ["plain", "native"])
def test_refusals(backend):
    from .test_native_host import make_ops
    ops = TorchOps() if backend == "plain" else make_ops()
    v = inputs(6, 16, 24)
    x, w, t, one = v["x"], v["w"], v["t"], torch.ones(6)
    for bad in (dict(x=x[None]), dict(w=w[:, :8]), dict(w=w.float()), dict(targets=t.int()), dict(targets=t[:5]), dict(targets=t.repeat(2)[::2]), dict(logit_scale=0.0),
                dict(logit_scale=float("nan")), dict(logit_scale=float("inf")), dict(w=w[:0])):
        with pytest.raises(ValueError):
            ops.linear_nll(**{"x": x, "w": w, "targets": t, **bad})
    good = dict(dloss=one, x=x, w=w, targets=t, loss=one, lse=one, dw_out=torch.empty_like(w))
    for bad in (dict(dloss=None), dict(dloss=one.double()), dict(dloss=one[:5]), dict(loss=one[:5]), dict(lse=torch.ones(12)[::2]), dict(dlse=one.bfloat16()), dict(dw_out=torch.empty(24, 16)),
                dict(dw_out=torch.empty_like(w)[:20])):
        with pytest.raises(ValueError):
            ops.linear_nll_bwd(**{**good, **bad})
    if backend == "native":
        with pytest.raises(ValueError, match="made for"):
            ops.linear_nll(x, w, t)
        ops.check_device = lambda t: None
        for bad in (dict(x=x.float(), w=w.float()), dict(x=x[:, :12].contiguous(), w=w[:, :12].contiguous()), dict(x=torch.empty(16, 6, dtype=torch.bfloat16).t()),
                    dict(w=torch.empty(24 * 16 + 1, dtype=torch.bfloat16)[1:].view(24, 16))):
            with pytest.raises(ValueError):
                ops.linear_nll(**{"x": x, "w": w, "targets": t, **bad})
        with pytest.raises(ValueError):
            ops.linear_nll_bwd(**{**good, "dw_out": torch.empty(16, 24, dtype=torch.bfloat16).t()})
        assert not ops.calls
    with pytest.raises(ValueError, match="memory of its own"):
        ops.linear_nll_bwd(**{**good, "dw_out": w})


# ------------------------------------------------------------------------------------------ kernels
@pytest.fixture(scope="module")
def native():
    from mini_trainer_b200.ops import get_ops
    return get_ops(torch.device("cuda:0"))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V", CASES + [(300, 2048, 4099), (1000, 1024, 32003), (257, 4096, 2048), (2, 256, 32000)])
@pytest.mark.parametrize("z,accumulate,scale", [(True, False, 1.0), (False, True, -0.3)])
def test_kernels(native, T, H, V, z, accumulate, scale):
    v = inputs(T, H, V, device="cuda", seed=V)
    torch.manual_seed(0)
    first = check(native, v, scale, z, accumulate)
    torch.manual_seed(0)
    again = check(native, v, scale, z, accumulate)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    native.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V", [(129, 64, 1500), (300, 1024, 4099), (40, 128, 513)])
def test_kernels_in_pieces(native, monkeypatch, T, H, V):
    """Many pieces, the last of them short: ``dx`` summed over them, each row of ``dw`` by its own."""
    v = inputs(T, H, V, device="cuda", seed=1)
    whole = check(native, v)
    monkeypatch.setattr(LN, "PIECE_BYTES", 1)
    monkeypatch.setattr(LN, "STATS_BYTES", 1)   # and the forward 256 tokens at a time
    assert LN.piece_columns(T, V) in (512, 256 * -(-V // (256 * -(-V // 512))))
    parts = check(native, v)
    assert torch.equal(whole[0], parts[0]) and torch.equal(whole[3], parts[3])
    check(native, v, 0.5, True, True)


@pytest.mark.gpu
def test_nearly_certain_targets(native):
    """A target with all but 1e-6 of the probability: its loss and the gradients, which are of that size, relative to themselves."""
    g = torch.Generator().manual_seed(5)
    w = (torch.randn(640, 256, generator=g) / 16).bfloat16()
    t = torch.randint(0, 640, (50,), generator=g)
    x = (w[t].float() * torch.linspace(10, 26, 50)[:, None]).bfloat16()
    logits = x.double() @ w.double().t()
    logp = torch.log_softmax(logits, 1).gather(1, t[:, None])[:, 0]
    assert (-logp).min() < 1e-6 < (-logp).median()
    x, w, t = x.cuda(), w.cuda(), t.cuda()
    loss, lse = native.linear_nll(x, w, t)
    D = (256 / 8 + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).amax(1).cpu()
    assert ((loss.cpu() + logp).abs() <= -logp * (2 * D + 2.0 ** -16 + 2.0 ** -21 * logits.abs().amax(1))).all()
    for i in range(0, 50, 7):   # a token alone, so that no other hides its gradient
        one = torch.ones(1, device="cuda")
        dw = torch.empty_like(w)
        dx = native.linear_nll_bwd(one, x[i:i + 1].contiguous(), w, t[i:i + 1].contiguous(), loss[i:i + 1].contiguous(), lse[i:i + 1].contiguous(), dw)
        p = torch.softmax(logits[i], 0)
        p[t[i].cpu()] = torch.expm1(logp[i])
        # U twice (operand and result), and D and what is beside it once per exponent
        tol = 2 * U + 2 * float(D[i]) + 2.0 ** -14
        assert float((dw.double().cpu() - p[:, None] * x[i].double().cpu()).norm() / (p.norm() * x[i].double().norm().cpu())) <= tol
        size = p.abs() @ w.double().cpu().abs()
        assert ((dx[0].double().cpu() - p @ w.double().cpu()).abs() <= tol * size).all()


@pytest.mark.gpu
def test_rows_that_are_not_counted_or_not_numbers(native):
    """An ignored row has no gradient whatever is upstream of it; logits that are not finite stay in their row of the losses and of ``dx``."""
    v = inputs(200, 64, 300, 0.5, device="cuda")
    ok = v["t"] != IGN
    v["dloss"][~ok] = float("nan")
    v["dlse"][~ok] = float("inf")
    loss, lse = native.linear_nll(v["x"], v["w"], v["t"])
    dw = torch.empty_like(v["w"])
    dx = native.linear_nll_bwd(v["dloss"], v["x"], v["w"], v["t"], loss, lse, dw, dlse=v["dlse"])
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and (dx[~ok] == 0).all()
    x = v["x"].clone()
    x[3], x[150, 5] = float("nan"), float("inf")
    l2, z2 = native.linear_nll(x, v["w"], v["t"])
    rest = torch.ones(200, dtype=torch.bool, device="cuda")
    rest[3] = rest[150] = False
    assert torch.equal(l2[rest], loss[rest]) and torch.equal(z2[rest], lse[rest]) and not torch.isfinite(z2[~rest]).any()
    dx2 = native.linear_nll_bwd(v["dloss"], x, v["w"], v["t"], l2, z2, dw, dlse=v["dlse"])
    assert torch.equal(dx2[rest], dx[rest])
    native.check_status()
    t = v["t"].clone()
    t[7], t[8] = 300, -1
    l3, _ = native.linear_nll(v["x"], v["w"], t)
    assert l3[7] == 0 and l3[8] == 0
    dx3 = native.linear_nll_bwd(torch.ones(200, device="cuda"), v["x"], v["w"], t, l3, lse, dw)
    assert (dx3[7:9] == 0).all()
    with pytest.raises(RuntimeError, match="target outside"):
        native.check_status()


def ignored_column(ops, device):
    """``ignore_index`` may be the number of a column (a padding token's): the column stays in every partition, its rows' too, which have no loss and no gradient."""
    v = inputs(60, 64, 300, 0.0, device=device)
    x, w, t = v["x"], v["w"], v["t"]
    t[::5] = 7
    ok = t != 7
    loss, lse = ops.linear_nll(x, w, t, ignore_index=7)
    every, same = ops.linear_nll(x, w, t)
    assert torch.equal(lse, same) and torch.equal(loss[ok], every[ok]) and (loss[~ok] == 0).all() and (every > 0).all()
    assert ((lse - torch.logsumexp(x.double() @ w.double().t(), 1)).abs() <= 1e-4).all()
    dw, dw2 = torch.empty_like(w), torch.empty_like(w)
    dx = ops.linear_nll_bwd(v["dloss"], x, w, t, loss, lse, dw, ignore_index=7, dlse=v["dlse"])
    weigh = torch.where(ok, v["dloss"], 0.0), torch.where(ok, v["dlse"], 0.0)
    want = ops.linear_nll_bwd(weigh[0], x, w, t, every, same, dw2, dlse=weigh[1])
    assert (dx[~ok] == 0).all() and torch.equal(dx, want) and torch.equal(dw, dw2)


def test_a_column_that_is_ignored():
    ignored_column(TorchOps(), "cpu")


@pytest.mark.gpu
def test_a_column_that_is_ignored_by_the_kernels(native):
    ignored_column(native, "cuda")
    native.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("piece", [None, 8192])
def test_captured_gradients_are_those_outside_of_a_graph(native, monkeypatch, piece):
    """Few tokens and many columns, whose sums over the vocabulary are divided: the same bits from every replay, whatever else runs beside it."""
    T, H, V = 64, 256, 30011
    if piece:
        monkeypatch.setattr(LN, "PIECE_BYTES", 2 * T * piece)
    v = inputs(T, H, V, device="cuda")
    dw = torch.empty_like(v["w"])

    def run(w):
        loss, lse = native.linear_nll(v["x"], v["w"], v["t"])
        return loss, lse, native.linear_nll_bwd(v["dloss"], v["x"], v["w"], v["t"], loss, lse, w, dlse=v["dlse"])
    want = run(dw)
    torch.cuda.synchronize()
    graph, captured = torch.cuda.CUDAGraph(), torch.empty_like(dw)
    with torch.cuda.graph(graph):
        got = run(captured)
    side, beside = torch.cuda.Stream(), torch.empty_like(dw)
    for _ in range(3):
        for t in (*got, captured):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = run(beside)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(captured, dw)
        assert all(torch.equal(a, b) for a, b in zip(other, want)) and torch.equal(beside, dw)
    v["dloss"].mul_(0.5), v["dlse"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    halves = run(dw)
    assert torch.equal(got[2], halves[2]) and torch.equal(captured, dw)
    native.check_status()


@pytest.mark.gpu
def test_no_tokens(native):
    w = torch.randn(24, 16, device="cuda").bfloat16()
    x, t, f = torch.empty(0, 16, dtype=torch.bfloat16, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, device="cuda")
    loss, lse = native.linear_nll(x, w, t)
    dw = torch.ones_like(w)
    assert native.linear_nll_bwd(f, x, w, t, loss, lse, dw, accumulate_dw=True).shape == (0, 16) and (dw == 1).all()
    native.linear_nll_bwd(f, x, w, t, loss, lse, dw)
    assert (dw == 0).all()


@pytest.mark.gpu
def test_under_capture_and_on_another_stream(native):
    v = inputs(300, 256, 5000, device="cuda")

    def run():
        loss, lse = native.linear_nll(v["x"], v["w"], v["t"])
        dw = torch.empty_like(v["w"])
        return loss, lse, native.linear_nll_bwd(v["dloss"], v["x"], v["w"], v["t"], loss, lse, dw, dlse=v["dlse"]), dw
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    want = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
    for a, b in zip(held[2:], want[2:]):   # products that split their reduction do not do so in a graph: other sums
        assert ((a.double() - b.double()).norm() <= 2 * U * b.double().norm())


@pytest.mark.gpu
def test_likelihoods_behind_2_31_logits(native):
    """Statistics, pieces and rows at offsets beyond 32 bits: the same tokens in front of many others."""
    T, H, V = 70000, 64, 40000
    v = inputs(300, H, V, device="cuda")
    x, t = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda"), torch.full((T,), IGN, device="cuda")
    x[-300:], t[-300:] = v["x"], v["t"]
    loss, lse = native.linear_nll(x, v["w"], t)
    l2, z2 = native.linear_nll(v["x"], v["w"], v["t"])
    assert torch.allclose(loss[-300:], l2, atol=1e-5) and torch.allclose(lse[-300:], z2, atol=1e-5)
    dl = torch.zeros(T, device="cuda")
    dl[-300:] = v["dloss"]
    dw, dw2 = torch.empty_like(v["w"]), torch.empty_like(v["w"])
    dx = native.linear_nll_bwd(dl, x, v["w"], t, loss, lse, dw)
    dx2 = native.linear_nll_bwd(v["dloss"], v["x"], v["w"], v["t"], l2, z2, dw2)
    for a, b in ((dx[-300:], dx2), (dw, dw2)):
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2 * U
    assert (dx[:-300] == 0).all()
